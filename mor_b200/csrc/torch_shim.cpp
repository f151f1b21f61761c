// Thin PyTorch front end over the C ABI of libmor_b200 (include/mor_b200.h).
//
// Registers the operator schemas of the reference extension verbatim
// (mor/csrc/fake_quantize.cpp:12-25 of boryiings/mor) under torch.ops.mor.*, for the
// CUDA dispatch key only -- there is no CPU implementation and none is wanted.  The
// shim validates arguments with TORCH_CHECK, allocates outputs and the workspace with
// torch::empty on the input's device, and launches on the CURRENT stream (the
// reference uses the legacy default stream).  It holds no arithmetic.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <vector>

#include "../../include/mor_b200.h"
#include "../../include/mor_b200_mx.h"

namespace mor {

namespace {

void* cur_stream() { return static_cast<void*>(at::cuda::getCurrentCUDAStream().stream()); }

void check_status(int rc, const char* op) {
    TORCH_CHECK(rc == MOR_B200_OK, "mor::", op, ": ", mor_b200_status_string(rc), " (status ", rc, ")");
}

int dtype_code(const at::Tensor& t, bool allow_fp32, const char* op) {
    if (t.dtype() == at::kBFloat16) return MOR_B200_BF16;
    TORCH_CHECK(allow_fp32 && t.dtype() == at::kFloat, "mor::", op, ": input must be bfloat16",
                allow_fp32 ? " or float32" : "");
    return MOR_B200_FP32;
}

at::Tensor checked_input(const at::Tensor& input, int64_t rows, int64_t cols, const char* op) {
    TORCH_CHECK(input.is_cuda(), "mor::", op, ": input must be a CUDA tensor");
    TORCH_CHECK(input.dim() == 2 && input.size(0) == rows && input.size(1) == cols, "mor::", op,
                ": input must be [dim_x, dim_y] = [", rows, ", ", cols, "]");
    return input.contiguous();
}

at::Tensor workspace(const at::Tensor& like, size_t bytes) {
    return torch::empty({(int64_t)bytes}, like.options().dtype(torch::kUInt8));
}

at::Tensor meta_tensor(const at::Tensor& like, int64_t rows, int64_t cols, int64_t br, int64_t bc) {
    const int64_t gx = (cols / 2 - 1) / (bc / 2) + 1, gy = (rows - 1) / br + 1;  // fake_quantize.cu:1757-1761
    return torch::empty({gy, gx}, like.options().dtype(torch::kInt32));
}

void check_fq_args(int64_t rows, int64_t cols, int64_t br, int64_t bc, int64_t sf_type) {
    TORCH_CHECK(rows > 0 && cols > 0 && br > 0 && bc >= 2, "mor::fake_quantize: sizes must be positive");
    TORCH_CHECK(cols % 2 == 0 && bc % 2 == 0, "mor::fake_quantize: dim_y and block_y must be even");
    TORCH_CHECK(sf_type == 1 || sf_type == 2, "mor::fake_quantize: sf_type must be 1 (fp32) or 2 (e8)");
}

// ---- fake_quantize ---------------------------------------------------------------
std::vector<at::Tensor> fake_quantize(const at::Tensor& input, int64_t rows, int64_t cols, int64_t br, int64_t bc,
                                      double clamp, int64_t mode, int64_t sf_type) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, "fake_quantize");
    const int dt = dtype_code(in, true, "fake_quantize");
    check_fq_args(rows, cols, br, bc, sf_type);
    at::Tensor out = torch::empty_like(in);
    at::Tensor meta = meta_tensor(in, rows, cols, br, bc);
    check_status(mor_b200_fake_quantize(in.data_ptr(), out.data_ptr(), meta.data_ptr<int32_t>(), dt, rows, cols,
                                        (int)br, (int)bc, clamp, (int)mode, (int)sf_type, cur_stream()),
                 "fake_quantize");
    return {out, meta};
}

at::Tensor fake_quantize_no_alloc(const at::Tensor& input, int64_t rows, int64_t cols, int64_t br, int64_t bc,
                                  double clamp, int64_t mode, int64_t sf_type, at::Tensor& result) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, "fake_quantize_no_alloc");
    const int dt = dtype_code(in, true, "fake_quantize_no_alloc");
    check_fq_args(rows, cols, br, bc, sf_type);
    TORCH_CHECK(result.is_cuda() && result.dtype() == in.dtype() && result.is_contiguous() && result.dim() == 2 &&
                    result.size(0) == rows && result.size(1) == cols,
                "mor::fake_quantize_no_alloc: result must be a contiguous CUDA tensor shaped and typed like input");
    at::Tensor meta = meta_tensor(in, rows, cols, br, bc);
    check_status(mor_b200_fake_quantize(in.data_ptr(), result.data_ptr(), meta.data_ptr<int32_t>(), dt, rows, cols,
                                        (int)br, (int)bc, clamp, (int)mode, (int)sf_type, cur_stream()),
                 "fake_quantize_no_alloc");
    return meta;
}

// ---- test operators ----------------------------------------------------------------
at::Tensor quant_dequant(const at::Tensor& input, int64_t rows, int64_t cols, int format, const char* op) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, op);
    TORCH_CHECK(in.dtype() == at::kFloat, "mor::", op, ": input must be float32");
    at::Tensor out = torch::empty_like(in);
    check_status(mor_b200_quant_dequant(in.data_ptr<float>(), out.data_ptr<float>(), rows, cols, format, cur_stream()), op);
    return out;
}
at::Tensor quant_dequant_e4m3(const at::Tensor& t, int64_t r, int64_t c, int64_t, int64_t) { return quant_dequant(t, r, c, MOR_B200_E4M3, "quant_dequant_e4m3"); }
at::Tensor quant_dequant_e5m2(const at::Tensor& t, int64_t r, int64_t c, int64_t, int64_t) { return quant_dequant(t, r, c, MOR_B200_E5M2, "quant_dequant_e5m2"); }
at::Tensor quant_dequant_e3m2(const at::Tensor& t, int64_t r, int64_t c, int64_t, int64_t) { return quant_dequant(t, r, c, MOR_B200_E3M2, "quant_dequant_e3m2"); }
at::Tensor quant_dequant_e2m3(const at::Tensor& t, int64_t r, int64_t c, int64_t, int64_t) { return quant_dequant(t, r, c, MOR_B200_E2M3, "quant_dequant_e2m3"); }

at::Tensor e8_scale(const at::Tensor& input, int64_t rows, int64_t cols, int rne, const char* op) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, op);
    TORCH_CHECK(in.dtype() == at::kFloat, "mor::", op, ": input must be float32");
    at::Tensor out = torch::empty_like(in);
    check_status(mor_b200_e4m3_with_e8_scale(in.data_ptr<float>(), out.data_ptr<float>(), rows, cols, rne, cur_stream()), op);
    return out;
}
at::Tensor e4m3_with_e8_scale_rne(const at::Tensor& t, int64_t r, int64_t c, int64_t, int64_t) { return e8_scale(t, r, c, 1, "e4m3_with_e8_scale_rne"); }
at::Tensor e4m3_with_e8_scale_rz(const at::Tensor& t, int64_t r, int64_t c, int64_t, int64_t) { return e8_scale(t, r, c, 0, "e4m3_with_e8_scale_rz"); }

// ---- block / channel scaling ---------------------------------------------------------
// Returns [out, meta, global_amax, global_non_zero, global_error]; inplace drops `out`.
// bf16 inputs report the non-zero count as int32 like the reference; float32 inputs
// (an extension for tensors of 2^31 elements and more) report int64.
std::vector<at::Tensor> scaling(int op, const char* name, at::Tensor in, at::Tensor out, int64_t rows, int64_t cols,
                                int64_t br, int64_t bc, double thr, int64_t ss) {
    const int dt = dtype_code(in, true, name);
    TORCH_CHECK(ss >= 1 && ss <= 4, "mor::", name, ": ss_mode must be 1..4");
    TORCH_CHECK(br > 0 && bc > 0 && rows % br == 0 && cols % bc == 0, "mor::", name,
                ": block shape must divide the tensor");
    if (op == MOR_B200_OP_CHANNEL_SCALING)
        TORCH_CHECK(br == 1 || bc == 1, "mor::", name, ": block_x or block_y must be 1");
    TORCH_CHECK(dt == MOR_B200_FP32 || rows * cols < (int64_t(1) << 31), "mor::", name,
                ": bfloat16 tensors report an int32 non-zero count; use float32 for 2^31 elements and more");
    const size_t wsb = mor_b200_workspace_bytes(op, rows, cols, (int)br, (int)bc);
    TORCH_CHECK(wsb > 0, "mor::", name, ": unsupported block shape ", br, " x ", bc);
    at::Tensor ws = workspace(in, wsb);
    auto iopt = in.options().dtype(torch::kInt32);
    auto fopt = in.options().dtype(torch::kFloat);
    at::Tensor meta = torch::empty({1}, iopt), gamax = torch::empty({1}, fopt), gerr = torch::empty({1}, fopt);
    const bool nnz64 = dt == MOR_B200_FP32;
    at::Tensor gnnz = torch::empty({1}, nnz64 ? in.options().dtype(torch::kInt64) : iopt);
    auto fn = op == MOR_B200_OP_BLOCK_SCALING ? mor_b200_block_scaling : mor_b200_channel_scaling;
    check_status(fn(in.data_ptr(), out.data_ptr(), dt, rows, cols, (int)br, (int)bc, thr, (int)ss,
                    meta.data_ptr<int32_t>(), gamax.data_ptr<float>(), gnnz.data_ptr(), nnz64 ? 1 : 0,
                    gerr.data_ptr<float>(), ws.data_ptr(), wsb, cur_stream()),
                 name);
    return {out, meta, gamax, gnnz, gerr};
}

std::vector<at::Tensor> fake_quantize_block_scaling(const at::Tensor& input, int64_t rows, int64_t cols, int64_t br,
                                                    int64_t bc, double thr, int64_t ss) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, "fake_quantize_block_scaling");
    return scaling(MOR_B200_OP_BLOCK_SCALING, "fake_quantize_block_scaling", in, torch::empty_like(in), rows, cols, br, bc, thr, ss);
}
std::vector<at::Tensor> fake_quantize_channel_scaling(const at::Tensor& input, int64_t rows, int64_t cols, int64_t br,
                                                      int64_t bc, double thr, int64_t ss) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, "fake_quantize_channel_scaling");
    return scaling(MOR_B200_OP_CHANNEL_SCALING, "fake_quantize_channel_scaling", in, torch::empty_like(in), rows, cols, br, bc, thr, ss);
}
std::vector<at::Tensor> scaling_inplace(int op, const char* name, at::Tensor& input, int64_t rows, int64_t cols,
                                        int64_t br, int64_t bc, double thr, int64_t ss) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, name);
    auto r = scaling(op, name, in, in, rows, cols, br, bc, thr, ss);
    if (!in.is_same(input)) input.copy_(in);  // a strided input was packed first
    return {r[1], r[2], r[3], r[4]};
}
std::vector<at::Tensor> fake_quantize_block_scaling_inplace(at::Tensor& input, int64_t rows, int64_t cols, int64_t br,
                                                            int64_t bc, double thr, int64_t ss) {
    return scaling_inplace(MOR_B200_OP_BLOCK_SCALING, "fake_quantize_block_scaling_inplace", input, rows, cols, br, bc, thr, ss);
}
std::vector<at::Tensor> fake_quantize_channel_scaling_inplace(at::Tensor& input, int64_t rows, int64_t cols,
                                                              int64_t br, int64_t bc, double thr, int64_t ss) {
    return scaling_inplace(MOR_B200_OP_CHANNEL_SCALING, "fake_quantize_channel_scaling_inplace", input, rows, cols, br, bc, thr, ss);
}

// ---- E8Mx -----------------------------------------------------------------------------
void e8mx_into(const at::Tensor& in, at::Tensor& out, int64_t rows, int64_t cols, int64_t qt, int64_t strat,
               const char* name) {
    TORCH_CHECK(in.dtype() == at::kBFloat16, "mor::", name, ": input must be bfloat16");
    TORCH_CHECK(qt >= 1 && qt <= 3, "mor::", name, ": quantize_type must be 1, 2 or 3");
    TORCH_CHECK(cols % 2 == 0, "mor::", name, ": dim_y must be even");
    const size_t wsb = mor_b200_workspace_bytes(MOR_B200_OP_E8MX, rows, cols, 0, 0);
    at::Tensor ws = workspace(in, wsb);
    check_status(mor_b200_e8mx(in.data_ptr(), out.data_ptr(), rows, cols, (int)qt, (int)strat, ws.data_ptr(), wsb,
                               cur_stream()),
                 name);
}
at::Tensor fake_quantize_e8mx(const at::Tensor& input, int64_t rows, int64_t cols, int64_t, int64_t, int64_t qt,
                              int64_t strat) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, "fake_quantize_e8mx");
    at::Tensor out = torch::empty_like(in);
    e8mx_into(in, out, rows, cols, qt, strat, "fake_quantize_e8mx");
    return out;
}
void fake_quantize_e8mx_inplace(const at::Tensor& input, int64_t rows, int64_t cols, int64_t, int64_t, int64_t qt,
                                int64_t strat, at::Tensor& result) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, "fake_quantize_e8mx_inplace");
    TORCH_CHECK(result.is_cuda() && result.dtype() == at::kBFloat16 && result.is_contiguous() && result.dim() == 2 &&
                    result.size(0) == rows && result.size(1) == cols,
                "mor::fake_quantize_e8mx_inplace: result must be a contiguous bfloat16 CUDA tensor shaped like input");
    e8mx_into(in, result, rows, cols, qt, strat, "fake_quantize_e8mx_inplace");
}

// ---- extension: per-group (MX) fake-quantize -------------------------------------------
// returns [out, scales]; scales is float32 [dim_x, dim_y / block_y]
std::vector<at::Tensor> fake_quantize_mx(const at::Tensor& input, int64_t rows, int64_t cols, int64_t bc,
                                         int64_t elem_format, int64_t sf_type) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, "fake_quantize_mx");
    const int dt = dtype_code(in, true, "fake_quantize_mx");
    TORCH_CHECK(bc > 0 && cols % bc == 0, "mor::fake_quantize_mx: block_y must divide dim_y");
    TORCH_CHECK(elem_format == MOR_B200_E4M3 || elem_format == MOR_B200_E5M2 || elem_format == MOR_B200_E2M3,
                "mor::fake_quantize_mx: elem_format must be 0 (E4M3), 1 (E5M2) or 3 (E2M3)");
    TORCH_CHECK(sf_type == 1 || sf_type == 2, "mor::fake_quantize_mx: sf_type must be 1 (fp32) or 2 (e8)");
    at::Tensor out = torch::empty_like(in);
    at::Tensor scales = torch::empty({rows, cols / bc}, in.options().dtype(torch::kFloat));
    check_status(mor_b200_fake_quantize_group(in.data_ptr(), out.data_ptr(), scales.data_ptr<float>(), dt, rows, cols,
                                              (int)bc, (int)elem_format, (int)sf_type, cur_stream()),
                 "fake_quantize_mx");
    return {out, scales};
}

// ---- extension: single-pass block scaling with a delayed tensor amax ---------------------
// returns [out, meta, amax of this tensor, non-zero count, error]; amax_in: float32[1] on the device
std::vector<at::Tensor> fake_quantize_block_scaling_delayed(const at::Tensor& input, int64_t rows, int64_t cols,
                                                            int64_t br, int64_t bc, double thr, int64_t ss,
                                                            const at::Tensor& amax_in) {
    const char* name = "fake_quantize_block_scaling_delayed";
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, name);
    const int dt = dtype_code(in, true, name);
    TORCH_CHECK(ss >= 1 && ss <= 4, "mor::", name, ": ss_mode must be 1..4");
    TORCH_CHECK(br == 128 && bc == 128 && rows % 128 == 0 && cols % 128 == 0, "mor::", name,
                ": 128 x 128 blocks that divide the tensor only");
    TORCH_CHECK(amax_in.is_cuda() && amax_in.scalar_type() == at::kFloat && amax_in.numel() == 1, "mor::", name,
                ": amax_in must be a float32 CUDA tensor with one element");
    TORCH_CHECK(dt == MOR_B200_FP32 || rows * cols < (int64_t(1) << 31), "mor::", name,
                ": bfloat16 tensors report an int32 non-zero count; use float32 for 2^31 elements and more");
    const size_t wsb = mor_b200_workspace_bytes(MOR_B200_OP_BLOCK_SCALING, rows, cols, 128, 128);
    at::Tensor ws = workspace(in, wsb);
    at::Tensor out = torch::empty_like(in);
    auto iopt = in.options().dtype(torch::kInt32);
    auto fopt = in.options().dtype(torch::kFloat);
    at::Tensor meta = torch::empty({1}, iopt), gamax = torch::empty({1}, fopt), gerr = torch::empty({1}, fopt);
    const bool nnz64 = dt == MOR_B200_FP32;
    at::Tensor gnnz = torch::empty({1}, nnz64 ? in.options().dtype(torch::kInt64) : iopt);
    check_status(mor_b200_block_scaling_delayed(in.data_ptr(), out.data_ptr(), dt, rows, cols, 128, 128, thr, (int)ss,
                                                amax_in.data_ptr<float>(), meta.data_ptr<int32_t>(),
                                                gamax.data_ptr<float>(), gnnz.data_ptr(), nnz64 ? 1 : 0,
                                                gerr.data_ptr<float>(), ws.data_ptr(), wsb, cur_stream()),
                 name);
    return {out, meta, gamax, gnnz, gerr};
}

// the same, and the result transposed as well: returns [out, out_t [dim_y, dim_x], meta, amax, non-zero count, error]
std::vector<at::Tensor> fake_quantize_block_scaling_delayed_t(const at::Tensor& input, int64_t rows, int64_t cols,
                                                              int64_t br, int64_t bc, double thr, int64_t ss,
                                                              const at::Tensor& amax_in) {
    const char* name = "fake_quantize_block_scaling_delayed_t";
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, name);
    const int dt = dtype_code(in, true, name);
    TORCH_CHECK(ss >= 1 && ss <= 4, "mor::", name, ": ss_mode must be 1..4");
    TORCH_CHECK(br == 128 && bc == 128 && rows % 128 == 0 && cols % 128 == 0, "mor::", name,
                ": 128 x 128 blocks that divide the tensor only");
    TORCH_CHECK(amax_in.is_cuda() && amax_in.scalar_type() == at::kFloat && amax_in.numel() == 1, "mor::", name,
                ": amax_in must be a float32 CUDA tensor with one element");
    TORCH_CHECK(dt == MOR_B200_FP32 || rows * cols < (int64_t(1) << 31), "mor::", name,
                ": bfloat16 tensors report an int32 non-zero count; use float32 for 2^31 elements and more");
    const size_t wsb = mor_b200_workspace_bytes(MOR_B200_OP_BLOCK_SCALING, rows, cols, 128, 128);
    at::Tensor ws = workspace(in, wsb);
    at::Tensor out = torch::empty_like(in);
    at::Tensor out_t = torch::empty({cols, rows}, in.options());
    auto iopt = in.options().dtype(torch::kInt32);
    auto fopt = in.options().dtype(torch::kFloat);
    at::Tensor meta = torch::empty({1}, iopt), gamax = torch::empty({1}, fopt), gerr = torch::empty({1}, fopt);
    const bool nnz64 = dt == MOR_B200_FP32;
    at::Tensor gnnz = torch::empty({1}, nnz64 ? in.options().dtype(torch::kInt64) : iopt);
    check_status(mor_b200_block_scaling_delayed_t(in.data_ptr(), out.data_ptr(), out_t.data_ptr(), dt, rows, cols, 128, 128,
                                                  thr, (int)ss, amax_in.data_ptr<float>(), meta.data_ptr<int32_t>(),
                                                  gamax.data_ptr<float>(), gnnz.data_ptr(), nnz64 ? 1 : 0,
                                                  gerr.data_ptr<float>(), ws.data_ptr(), wsb, cur_stream()),
                 name);
    return {out, out_t, meta, gamax, gnnz, gerr};
}

// ---- extension: real quantized output (codes + E8M0 scale bytes) -----------------------
// returns [payload uint8 [dim_x, dim_y], scales uint8 [dim_x, dim_y / block_y]]
std::vector<at::Tensor> quantize_mx(const at::Tensor& input, int64_t rows, int64_t cols, int64_t bc, int64_t elem_format, bool operand) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, "quantize_mx");
    if (reinterpret_cast<uintptr_t>(in.data_ptr()) % 16) in = in.clone();   // a slice of a longer tensor
    TORCH_CHECK(in.scalar_type() == at::kBFloat16, "mor::quantize_mx: bfloat16 input only");
    TORCH_CHECK(bc > 0 && cols % bc == 0, "mor::quantize_mx: block_y must divide dim_y");
    TORCH_CHECK(elem_format == MOR_B200_E4M3 || elem_format == MOR_B200_E5M2 || elem_format == MOR_B200_E2M3,
                "mor::quantize_mx: elem_format must be 0 (E4M3), 1 (E5M2) or 3 (E2M3)");
    at::Tensor payload = torch::empty({rows, cols}, in.options().dtype(torch::kUInt8));
    at::Tensor scales = torch::empty({rows, cols / bc}, in.options().dtype(torch::kUInt8));
    if (rows == 0) return {payload, scales};
    check_status(mor_b200_quantize_mx(in.data_ptr(), payload.data_ptr(), scales.data_ptr(), rows, cols, (int)bc,
                                      (int)elem_format + (operand ? MOR_B200_MX_OPERAND : 0), cur_stream()),
                 "quantize_mx");
    return {payload, scales};
}

// returns [payload uint8 [dim_x, dim_y * 3 / 4] (E2M3, six bits per element), scales uint8 [dim_x, dim_y / block_y]]
std::vector<at::Tensor> quantize_mx_fp6(const at::Tensor& input, int64_t rows, int64_t cols, int64_t bc) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, "quantize_mx_fp6");
    TORCH_CHECK(in.scalar_type() == at::kBFloat16, "mor::quantize_mx_fp6: bfloat16 input only");
    TORCH_CHECK(bc > 0 && cols % bc == 0 && cols % 8 == 0, "mor::quantize_mx_fp6: block_y must divide dim_y, dim_y a multiple of 8");
    at::Tensor payload = torch::empty({rows, cols * 3 / 4}, in.options().dtype(torch::kUInt8));
    at::Tensor scales = torch::empty({rows, cols / bc}, in.options().dtype(torch::kUInt8));
    check_status(mor_b200_quantize_mx_fp6(in.data_ptr(), payload.data_ptr(), scales.data_ptr(), rows, cols, (int)bc,
                                          cur_stream()),
                 "quantize_mx_fp6");
    return {payload, scales};
}

// returns [payload uint8 [dim_x, dim_y] (E4M3 bytes), scales float32 [dim_x / block_x, dim_y / block_y], global_amax float32[1]]
std::vector<at::Tensor> quantize_scaled(const at::Tensor& input, int64_t rows, int64_t cols, int64_t br, int64_t bc,
                                        int64_t ss) {
    const c10::cuda::CUDAGuard guard(input.device());
    at::Tensor in = checked_input(input, rows, cols, "quantize_scaled");
    const int dt = dtype_code(in, true, "quantize_scaled");
    TORCH_CHECK(ss == 1 || ss == 3 || ss == 4, "mor::quantize_scaled: ss_mode must be 1, 3 or 4 (binary32 scales)");
    TORCH_CHECK(br > 0 && bc > 0 && rows % br == 0 && cols % bc == 0, "mor::quantize_scaled: block shape must divide the tensor");
    const int op = (br == 1 || bc == 1) ? MOR_B200_OP_CHANNEL_SCALING : MOR_B200_OP_BLOCK_SCALING;
    const size_t wsb = mor_b200_workspace_bytes(op, rows, cols, (int)br, (int)bc);
    TORCH_CHECK(wsb > 0, "mor::quantize_scaled: unsupported block shape ", br, " x ", bc);
    at::Tensor ws = workspace(in, wsb);
    at::Tensor payload = torch::empty({rows, cols}, in.options().dtype(torch::kUInt8));
    at::Tensor scales = torch::empty({rows / br, cols / bc}, in.options().dtype(torch::kFloat));
    at::Tensor gamax = torch::empty({1}, in.options().dtype(torch::kFloat));
    check_status(mor_b200_quantize_scaled(in.data_ptr(), payload.data_ptr(), scales.data_ptr<float>(), dt, rows, cols, (int)br,
                                          (int)bc, (int)ss, nullptr, gamax.data_ptr<float>(), ws.data_ptr(), wsb, cur_stream()),
                 "quantize_scaled");
    return {payload, scales, gamax};
}

// ---- extension: microscaled operands (include/mor_b200_mx.h) -----------------------------
// One code per element, or two to a byte for E2M1; the tensors of one operand lie on one device.
// Outputs of these operators are taken from the allocator directly: the calls for single tokens are as long as their host side.
at::Tensor mx_empty(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt));
}
bool mx_format_ok(int64_t f) { return f == MOR_B200_E4M3 || f == MOR_B200_E5M2 || f == MOR_B200_E2M3 || f == MOR_B200_MX_E2M1; }

at::Tensor mx_part(const at::Tensor& t, int64_t rows, int64_t cols, const at::Tensor& like, size_t align, const char* op, const char* what) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), "mor::", op, ": ", what, " must be on ", like.device());
    TORCH_CHECK(t.scalar_type() == at::kByte, "mor::", op, ": ", what, " must be uint8");
    TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, "mor::", op, ": ", what, " must be [", rows, ", ", cols, "]");
    at::Tensor c = t.contiguous();
    if (reinterpret_cast<uintptr_t>(c.data_ptr()) % align) c = c.clone();
    return c;
}
at::Tensor mx_payload(const at::Tensor& t, int64_t rows, int64_t cols, int64_t format, const at::Tensor& like, const char* op, const char* what) {
    return mx_part(t, rows, format == MOR_B200_MX_E2M1 ? cols / 2 : cols, like, 16, op, what);
}
// rows as they are where the copy engine can take them (unit stride along a row, rows a multiple of 16 bytes apart), packed otherwise
at::Tensor mx_rows(const at::Tensor& t, int64_t& pitch) {
    const int64_t w = t.element_size(), packed = (t.size(1) * w + 15) / 16 * 16 / w;
    pitch = t.size(0) > 1 ? t.stride(0) : packed;
    const bool unit = t.stride(1) == 1 || t.size(1) == 1;
    if (unit && pitch >= t.size(1) && pitch * w % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0) return t;
    pitch = packed;
    at::Tensor p = mx_empty({t.size(0), packed}, t.scalar_type(), t);
    p.narrow(1, 0, t.size(1)).copy_(t);
    return p;
}

at::Tensor column_sums(const at::Tensor& input, int64_t rows, int64_t cols) {
    TORCH_CHECK(input.is_cuda(), "mor::column_sums: input must be a CUDA tensor");
    const c10::cuda::CUDAGuard guard(input.device());
    TORCH_CHECK(input.dim() == 2 && input.size(0) == rows && input.size(1) == cols, "mor::column_sums: input must be [dim_x, dim_y] = [",
                rows, ", ", cols, "]");
    TORCH_CHECK(input.scalar_type() == at::kBFloat16, "mor::column_sums: input must be bfloat16");
    at::Tensor out = mx_empty({cols}, at::kBFloat16, input);
    int64_t pitch = 0;
    at::Tensor in = mx_rows(input, pitch);
    check_status(mor_b200_mx_column_sums(in.data_ptr(), pitch, rows, cols, out.data_ptr(), cur_stream()), "column_sums");
    return out;
}

// returns [payload uint8 [dim_x, dim_y / 2], scales uint8 [dim_x, dim_y / 32]]
std::vector<at::Tensor> quantize_mx_fp4(const at::Tensor& input, int64_t rows, int64_t cols, int64_t bc) {
    TORCH_CHECK(input.is_cuda(), "mor::quantize_mx_fp4: input must be a CUDA tensor");
    const c10::cuda::CUDAGuard guard(input.device());
    TORCH_CHECK(input.dim() == 2 && input.size(0) == rows && input.size(1) == cols,
                "mor::quantize_mx_fp4: input must be [dim_x, dim_y] = [", rows, ", ", cols, "]");
    const int dt = dtype_code(input, true, "quantize_mx_fp4");
    TORCH_CHECK(bc == 32, "mor::quantize_mx_fp4: block_y must be 32");
    TORCH_CHECK(cols > 0 && cols % 32 == 0, "mor::quantize_mx_fp4: dim_y must be a positive multiple of 32");
    at::Tensor payload = mx_empty({rows, cols / 2}, at::kByte, input);
    at::Tensor scales = mx_empty({rows, cols / 32}, at::kByte, input);
    if (rows == 0) return {payload, scales};
    int64_t pitch = 0;
    at::Tensor in = mx_rows(input, pitch);
    check_status(mor_b200_mx_quantize_fp4(in.data_ptr(), dt, rows, cols, pitch, payload.data_ptr(), scales.data_ptr(), cur_stream()),
                 "quantize_mx_fp4");
    return {payload, scales};
}

at::Tensor dequantize_mx(const at::Tensor& payload, const at::Tensor& scales, int64_t rows, int64_t cols, int64_t bc, int64_t format,
                         at::ScalarType dtype) {
    TORCH_CHECK(payload.is_cuda(), "mor::dequantize_mx: payload must be a CUDA tensor");
    const c10::cuda::CUDAGuard guard(payload.device());
    TORCH_CHECK(mx_format_ok(format), "mor::dequantize_mx: elem_format must be 0 (E4M3), 1 (E5M2), 3 (E2M3) or 4 (E2M1)");
    TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kFloat, "mor::dequantize_mx: out_dtype must be bfloat16 or float32");
    TORCH_CHECK(rows >= 0 && cols > 0 && bc >= 8 && bc <= 256 && (bc & (bc - 1)) == 0 && cols % bc == 0,
                "mor::dequantize_mx: block_y must be a power of two from 8 to 256 that divides dim_y");
    at::Tensor p = mx_payload(payload, rows, cols, format, payload, "dequantize_mx", "payload");
    at::Tensor s = mx_part(scales, rows, cols / bc, payload, 1, "dequantize_mx", "scales");
    at::Tensor out = mx_empty({rows, cols}, dtype, payload);
    check_status(mor_b200_mx_dequantize(p.data_ptr(), s.data_ptr(), out.data_ptr(), dtype == at::kFloat ? MOR_B200_FP32 : MOR_B200_BF16,
                                        rows, cols, (int)bc, (int)format, cur_stream()),
                 "dequantize_mx");
    return out;
}

at::Tensor mx_matmul(const at::Tensor& a, const at::Tensor& a_scales, const at::Tensor& b, const at::Tensor& b_scales, int64_t m, int64_t n,
                     int64_t k, int64_t a_format, int64_t b_format, const std::optional<at::Tensor>& bias) {
    TORCH_CHECK(a.is_cuda(), "mor::mx_matmul: a must be a CUDA tensor");
    const c10::cuda::CUDAGuard guard(a.device());
    const bool fp4 = a_format == MOR_B200_MX_E2M1 && b_format == MOR_B200_MX_E2M1;
    const bool fp8 = (a_format == MOR_B200_E4M3 || a_format == MOR_B200_E5M2) && (b_format == MOR_B200_E4M3 || b_format == MOR_B200_E5M2);
    TORCH_CHECK(fp4 || fp8, "mor::mx_matmul: formats must be 4 and 4 (E2M1), or each 0 (E4M3) or 1 (E5M2)");
    TORCH_CHECK(m >= 0 && n >= 0 && k > 0 && k % 32 == 0, "mor::mx_matmul: dim_k must be a positive multiple of 32");
    at::Tensor ac = mx_payload(a, m, k, a_format, a, "mx_matmul", "a"), as = mx_part(a_scales, m, k / 32, a, 16, "mx_matmul", "a_scales");
    at::Tensor bcod = mx_payload(b, n, k, b_format, a, "mx_matmul", "b"), bs = mx_part(b_scales, n, k / 32, a, 16, "mx_matmul", "b_scales");
    at::Tensor bi;
    if (bias.has_value() && bias->defined()) {
        TORCH_CHECK(bias->is_cuda() && bias->device() == a.device() && bias->scalar_type() == at::kBFloat16 && bias->dim() == 1 && bias->size(0) == n,
                    "mor::mx_matmul: bias must be bfloat16 [dim_n] on ", a.device());
        bi = bias->contiguous();
    }
    at::Tensor out = mx_empty({m, n}, at::kBFloat16, a);
    const size_t wsb = mor_b200_mx_matmul_workspace_bytes(m, n, k, (int)a_format);
    at::Tensor ws;
    if (wsb) ws = mx_empty({(int64_t)wsb}, at::kByte, a);
    check_status(mor_b200_mx_matmul(ac.data_ptr(), as.data_ptr(), bcod.data_ptr(), bs.data_ptr(), m, n, k, (int)a_format, (int)b_format,
                                    bi.defined() ? bi.data_ptr() : nullptr, out.data_ptr(), wsb ? ws.data_ptr() : nullptr, wsb, cur_stream()),
                 "mx_matmul");
    return out;
}

at::Tensor mx_matmul_grad(const at::Tensor& g, const at::Tensor& payload, const at::Tensor& scales, int64_t m, int64_t n, int64_t k,
                          int64_t format, bool transpose_g) {
    TORCH_CHECK(g.is_cuda(), "mor::mx_matmul_grad: g must be a CUDA tensor");
    const c10::cuda::CUDAGuard guard(g.device());
    TORCH_CHECK(mx_format_ok(format), "mor::mx_matmul_grad: elem_format must be 0 (E4M3), 1 (E5M2), 3 (E2M3) or 4 (E2M1)");
    TORCH_CHECK(m >= 0 && n >= 0 && k >= 0 && n % 32 == 0, "mor::mx_matmul_grad: dim_n must be a multiple of 32");
    TORCH_CHECK(g.scalar_type() == at::kBFloat16, "mor::mx_matmul_grad: g must be bfloat16");
    TORCH_CHECK(g.dim() == 2 && g.size(0) == (transpose_g ? k : m) && g.size(1) == (transpose_g ? m : k),
                "mor::mx_matmul_grad: g must be [dim_m, dim_k], or [dim_k, dim_m] with transpose_g");
    at::Tensor p = mx_payload(payload, k, n, format, g, "mx_matmul_grad", "payload");
    at::Tensor s = mx_part(scales, k, n / 32, g, 1, "mx_matmul_grad", "scales");
    at::Tensor out = mx_empty({m, n}, at::kBFloat16, g);
    if (m == 0 || n == 0) return out;
    int64_t pitch = 0;
    at::Tensor gr = mx_rows(g, pitch);
    check_status(mor_b200_mx_matmul_grad(gr.data_ptr(), pitch, p.data_ptr(), s.data_ptr(), m, n, k, (int)format, transpose_g ? 1 : 0,
                                         out.data_ptr(), cur_stream()),
                 "mx_matmul_grad");
    return out;
}

// ---- a linear layer on microscaled operands -----------------------------------------------
// Codes and scale bytes of a [rows, cols] tensor in groups of 32 columns.
std::vector<at::Tensor> mx_quantized(const at::Tensor& x, int64_t format) {
    const int64_t r = x.size(0), c = x.size(1);
    if (format == MOR_B200_MX_E2M1) return quantize_mx_fp4(x, r, c, 32);
    TORCH_CHECK(x.scalar_type() == at::kBFloat16 && c > 0 && c % 32 == 0,
                "mor::mx_linear: 8-bit operands are quantised from bfloat16, with a width that is a positive multiple of 32");
    return quantize_mx(x, r, c, 32, format, /*operand=*/true);
}

// A layer's bias as the product adds it: in binary32 before the result's rounding, from bf16, the result's own precision.
std::optional<at::Tensor> mx_bias(const std::optional<at::Tensor>& bias) {
    if (!bias.has_value() || !bias->defined() || bias->scalar_type() == at::kBFloat16) return bias;
    return bias->to(at::kBFloat16);
}

// [tokens, n] in the shape of x but for its last dimension.  Not a view that autograd tracks: it is the only tensor on its memory, and
// as a view made inside a custom function, or without gradients, it could not be written in place (relu_, y += ...).
at::Tensor mx_shaped(const at::Tensor& y, at::IntArrayRef x_sizes) {
    if (x_sizes.size() == 2) return y;
    std::vector<int64_t> shape = x_sizes.vec();
    shape.back() = y.size(1);
    return at::_unsafe_view(y, shape);
}

// Straight-through: the gradients are those of a linear layer fed the quantised values, computed from the codes, which are
// all that the forward pass keeps of the input and the weight.  The operators inside are called as functions, past the
// dispatcher, which would cost each of seven calls a few microseconds: dispatch modes, tracing and profiles by operator see
// mx_linear (mx_linear_packed) alone.
struct MxLinear : public torch::autograd::Function<MxLinear> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                              const std::optional<at::Tensor>& bias, int64_t format) {
        const int64_t k = weight.size(1), n = weight.size(0);
        at::Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, k});
        const int64_t m = x2.size(0);
        const std::vector<at::Tensor> xq = mx_quantized(x2, format), wq = mx_quantized(weight, format);
        const std::optional<at::Tensor> b = mx_bias(bias);
        at::Tensor y = mx_matmul(xq[0], xq[1], wq[0], wq[1], m, n, k, format, format, b);
        const bool need_x = x.requires_grad(), need_w = weight.requires_grad();
        ctx->save_for_backward({need_x ? wq[0] : at::Tensor(), need_x ? wq[1] : at::Tensor(), need_w ? xq[0] : at::Tensor(),
                                need_w ? xq[1] : at::Tensor()});
        ctx->saved_data["format"] = format;
        ctx->saved_data["x_sizes"] = x.sizes().vec();
        ctx->saved_data["n"] = n;
        ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)x.scalar_type(), (int64_t)weight.scalar_type(),
                                                        b.has_value() && b->defined() ? (int64_t)bias->scalar_type() : 0};
        return mx_shaped(y, x.sizes());
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "mor::mx_linear is differentiable once: its gradients have no gradient (create_graph)");
        const torch::autograd::variable_list kept = ctx->get_saved_variables();
        const int64_t format = ctx->saved_data["format"].toInt(), n = ctx->saved_data["n"].toInt();
        const std::vector<int64_t> sizes = ctx->saved_data["x_sizes"].toIntVector(), types = ctx->saved_data["types"].toIntVector();
        const int64_t k = sizes.back();
        int64_t m = 1;   // counted, since a layer of no outputs leaves nothing to infer it from
        for (size_t i = 0; i + 1 < sizes.size(); ++i) m *= sizes[i];
        at::Tensor g = grads[0].dim() == 2 ? grads[0] : grads[0].reshape({m, n});
        int64_t pitch = 0;
        g = mx_rows(g, pitch).narrow(1, 0, n);   // packed once where its rows do not fit, for all that read it
        auto typed = [](at::Tensor t, int64_t type) { return t.scalar_type() == (at::ScalarType)type ? t : t.to((at::ScalarType)type); };
        at::Tensor gx, gw, gb;
        // a gradient that this pass does not ask for costs a whole product
        if (kept[0].defined() && ctx->needs_input_grad(0)) {
            gx = typed(mx_matmul_grad(g, kept[0], kept[1], m, k, n, format, false), types[0]);
            if (sizes.size() != 2) gx = gx.reshape(sizes);
        }
        if (kept[2].defined() && ctx->needs_input_grad(1)) gw = typed(mx_matmul_grad(g, kept[2], kept[3], n, k, m, format, true), types[1]);
        if (types[2] && ctx->needs_input_grad(2)) gb = typed(column_sums(g, m, n), types[2]);
        return {gx, gw, gb, at::Tensor()};
    }
};

at::Tensor mx_linear(const at::Tensor& x, const at::Tensor& weight, const std::optional<at::Tensor>& bias, int64_t format) {
    TORCH_CHECK(x.is_cuda() && weight.device() == x.device(), "mor::mx_linear: x and weight must be CUDA tensors on one device");
    TORCH_CHECK(format == MOR_B200_E4M3 || format == MOR_B200_E5M2 || format == MOR_B200_MX_E2M1,
                "mor::mx_linear: elem_format must be 0 (E4M3), 1 (E5M2) or 4 (E2M1)");
    TORCH_CHECK(weight.dim() == 2 && x.dim() >= 1 && x.size(-1) == weight.size(1), "mor::mx_linear: x must be [..., in] and weight [out, in]");
    return MxLinear::apply(x, weight, bias, format);
}

// The forward pass alone, from weights that were quantised once.
at::Tensor mx_linear_packed(const at::Tensor& x, const at::Tensor& payload, const at::Tensor& scales, const std::optional<at::Tensor>& bias,
                            int64_t format) {
    TORCH_CHECK(x.is_cuda(), "mor::mx_linear_packed: x must be a CUDA tensor");
    TORCH_CHECK(format == MOR_B200_E4M3 || format == MOR_B200_E5M2 || format == MOR_B200_MX_E2M1,
                "mor::mx_linear_packed: elem_format must be 0 (E4M3), 1 (E5M2) or 4 (E2M1)");
    TORCH_CHECK(payload.dim() == 2 && x.dim() >= 1, "mor::mx_linear_packed: x must be [..., in] and payload that of [out, in]");
    const at::NoGradGuard none;
    const int64_t k = x.size(-1), n = payload.size(0);
    at::Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, k});
    const std::vector<at::Tensor> q = mx_quantized(x2, format);
    at::Tensor y = mx_matmul(q[0], q[1], payload, scales, x2.size(0), n, k, format, format, mx_bias(bias));
    return mx_shaped(y, x.sizes());
}

}  // namespace

// Registers _C as a Python extension module.
PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {}

TORCH_LIBRARY(mor, m) {
  // the fourteen schemas of the reference, unchanged
  m.def("fake_quantize(Tensor input, int dim_x, int dim_y, int block_x, int block_y, float clamp_threshold, int mode, int sf_type) -> Tensor[]");
  m.def("fake_quantize_no_alloc(Tensor input, int dim_x, int dim_y, int block_x, int block_y, float clamp_threshold, int mode, int sf_type, Tensor result) -> Tensor");
  m.def("quant_dequant_e4m3(Tensor input, int dim_x, int dim_y, int block_x, int block_y) -> Tensor");
  m.def("quant_dequant_e5m2(Tensor input, int dim_x, int dim_y, int block_x, int block_y) -> Tensor");
  m.def("quant_dequant_e3m2(Tensor input, int dim_x, int dim_y, int block_x, int block_y) -> Tensor");
  m.def("quant_dequant_e2m3(Tensor input, int dim_x, int dim_y, int block_x, int block_y) -> Tensor");
  m.def("e4m3_with_e8_scale_rne(Tensor input, int dim_x, int dim_y, int block_x, int block_y) -> Tensor");
  m.def("e4m3_with_e8_scale_rz(Tensor input, int dim_x, int dim_y, int block_x, int block_y) -> Tensor");
  m.def("fake_quantize_block_scaling(Tensor input, int dim_x, int dim_y, int block_x, int block_y, float e4m3_threshold, int ss_mode) -> Tensor[]");
  m.def("fake_quantize_block_scaling_inplace(Tensor input, int dim_x, int dim_y, int block_x, int block_y, float e4m3_threshold, int ss_mode) -> Tensor[]");
  m.def("fake_quantize_e8mx(Tensor input, int dim_x, int dim_y, int block_x, int block_y, int quantize_type, int scaling_strategy) -> Tensor");
  m.def("fake_quantize_e8mx_inplace(Tensor input, int dim_x, int dim_y, int block_x, int block_y, int quantize_type, int scaling_strategy, Tensor result) -> ()");
  m.def("fake_quantize_channel_scaling(Tensor input, int dim_x, int dim_y, int block_x, int block_y, float e4m3_threshold, int ss_mode) -> Tensor[]");
  m.def("fake_quantize_channel_scaling_inplace(Tensor input, int dim_x, int dim_y, int block_x, int block_y, float e4m3_threshold, int ss_mode) -> Tensor[]");
  // addition: one scale per 1 x block_y group (MX), E4M3 / E5M2 / E2M3 elements
  m.def("fake_quantize_mx(Tensor input, int dim_x, int dim_y, int block_y, int elem_format, int sf_type) -> Tensor[]");
  m.def("quantize_mx(Tensor input, int dim_x, int dim_y, int block_y, int elem_format, bool operand=False) -> Tensor[]");
  m.def("quantize_mx_fp6(Tensor input, int dim_x, int dim_y, int block_y) -> Tensor[]");
  m.def("quantize_scaled(Tensor input, int dim_x, int dim_y, int block_x, int block_y, int ss_mode) -> Tensor[]");
  m.def("fake_quantize_block_scaling_delayed(Tensor input, int dim_x, int dim_y, int block_x, int block_y, float e4m3_threshold, int ss_mode, Tensor amax_in) -> Tensor[]");
  m.def("fake_quantize_block_scaling_delayed_t(Tensor input, int dim_x, int dim_y, int block_x, int block_y, float e4m3_threshold, int ss_mode, Tensor amax_in) -> Tensor[]");
  // microscaled operands: 4-bit codes, codes back to values, products
  m.def("quantize_mx_fp4(Tensor input, int dim_x, int dim_y, int block_y) -> Tensor[]");
  m.def("dequantize_mx(Tensor payload, Tensor scales, int dim_x, int dim_y, int block_y, int elem_format, ScalarType out_dtype) -> Tensor");
  m.def("mx_matmul(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, int dim_m, int dim_n, int dim_k, int a_format, int b_format, Tensor? bias) -> Tensor");
  m.def("mx_matmul_grad(Tensor g, Tensor payload, Tensor scales, int dim_m, int dim_n, int dim_k, int elem_format, bool transpose_g) -> Tensor");
  m.def("column_sums(Tensor input, int dim_x, int dim_y) -> Tensor");
  m.def("mx_linear(Tensor x, Tensor weight, Tensor? bias, int elem_format) -> Tensor", &mx_linear);   // composed of the above, with its gradient
  m.def("mx_linear_packed(Tensor x, Tensor payload, Tensor scales, Tensor? bias, int elem_format) -> Tensor", &mx_linear_packed);
}

TORCH_LIBRARY_IMPL(mor, CUDA, m) {
  m.impl("fake_quantize", &fake_quantize);
  m.impl("fake_quantize_no_alloc", &fake_quantize_no_alloc);
  m.impl("quant_dequant_e4m3", &quant_dequant_e4m3);
  m.impl("quant_dequant_e5m2", &quant_dequant_e5m2);
  m.impl("quant_dequant_e3m2", &quant_dequant_e3m2);
  m.impl("quant_dequant_e2m3", &quant_dequant_e2m3);
  m.impl("e4m3_with_e8_scale_rne", &e4m3_with_e8_scale_rne);
  m.impl("e4m3_with_e8_scale_rz", &e4m3_with_e8_scale_rz);
  m.impl("fake_quantize_block_scaling", &fake_quantize_block_scaling);
  m.impl("fake_quantize_block_scaling_inplace", &fake_quantize_block_scaling_inplace);
  m.impl("fake_quantize_e8mx", &fake_quantize_e8mx);
  m.impl("fake_quantize_e8mx_inplace", &fake_quantize_e8mx_inplace);
  m.impl("fake_quantize_channel_scaling", &fake_quantize_channel_scaling);
  m.impl("fake_quantize_channel_scaling_inplace", &fake_quantize_channel_scaling_inplace);
  m.impl("fake_quantize_mx", &fake_quantize_mx);
  m.impl("quantize_mx", &quantize_mx);
  m.impl("quantize_mx_fp6", &quantize_mx_fp6);
  m.impl("quantize_scaled", &quantize_scaled);
  m.impl("fake_quantize_block_scaling_delayed", &fake_quantize_block_scaling_delayed);
  m.impl("fake_quantize_block_scaling_delayed_t", &fake_quantize_block_scaling_delayed_t);
  m.impl("quantize_mx_fp4", &quantize_mx_fp4);
  m.impl("column_sums", &column_sums);
  m.impl("dequantize_mx", &dequantize_mx);
  m.impl("mx_matmul", &mx_matmul);
  m.impl("mx_matmul_grad", &mx_matmul_grad);
}

}  // namespace mor
