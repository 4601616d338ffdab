// tinym_torch_op.cpp -- torch custom-op shim over the C ABI.
//
// Registers the reference's op namespace and schema
// (src/torch_candidate_extension.cu:85-91):
//     sm120_fp8_gemm::run(Tensor a, Tensor b, float alpha) -> Tensor
// plus a device-alpha form used by candidate_kernel.fp8_gemm:
//     sm120_fp8_gemm::run_alpha_tensor(Tensor a, Tensor b, Tensor alpha) -> Tensor
// and the packed-weight pair behind candidate_kernel.prepare_weights'
// optional repack (tinym_pack_weights / tinym_fp8_gemm_packed):
//     sm120_fp8_gemm::pack_weights(Tensor b) -> Tensor            (uint8, packed layout)
//     sm120_fp8_gemm::run_packed(Tensor a, Tensor b_packed, int n, int k, Tensor alpha) -> Tensor
// and the fused activation path (tinym_fp8_gemm_quant_act): a BF16 / FP32
// activation quantised per tensor on the device, then the GEMM:
//     sm120_fp8_gemm::run_quant_act(Tensor x, Tensor b, Tensor w_scale) -> (Tensor y, Tensor x_scale)
// and the operators with no counterpart in the reference (include/tinym_b200.h):
// run_grouped (one weight per group of rows), mxfp4_quantize /
// mxfp4_dequantize, run_mxfp4 and run_mxfp4_grouped; the *_out forms write
// into the caller's Y and leave rows of no group as they were.
// Input checks mirror check_inputs (src/torch_candidate_extension.cu:17-31)
// and raise the same RuntimeError (TORCH_CHECK) messages; every op also
// raises before launching if an earlier GEMM on the device ran out of a
// bounded wait (tinym_pending_errors).  Shape support is
// decided by the C ABI (1 <= M <= 16, K % 16 == 0) instead of the six-point
// gate of :40-46.  Y is allocated by the op (as in :49-50) and the kernel is
// launched on the current stream of A's device (:48,:57).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/util/Exception.h>
#include <torch/library.h>

#include <cmath>
#include <string>

#include "../../include/tinym_b200.h"

namespace {

// Numbers go into messages as text: formatting them through the message's
// stream crashes where the compiler's libstdc++ is not the one loaded.
std::string num(int64_t v) { return std::to_string(v); }

void check_inputs(const at::Tensor& a, const at::Tensor& b) {
    TORCH_CHECK(a.is_cuda() && b.is_cuda(), "A and B must be CUDA tensors");
    TORCH_CHECK(a.get_device() == b.get_device(), "A and B must be on the same CUDA device");
    TORCH_CHECK(a.dim() == 2 && b.dim() == 2, "A and B must both be rank-2 tensors");
    TORCH_CHECK(a.is_contiguous() && b.is_contiguous(), "A and B must be contiguous row-major tensors");
    TORCH_CHECK(a.scalar_type() == at::ScalarType::Float8_e4m3fn &&
                    b.scalar_type() == at::ScalarType::Float8_e4m3fn,
                "A and B must have dtype torch.float8_e4m3fn");
    TORCH_CHECK(a.size(1) == b.size(1), "A and B must have the same K dimension");
}

void raise_status(int st) {
    TORCH_CHECK(st == TINYM_OK, tinym_status_string(st), ": ", tinym_last_error());
}

// A GEMM whose bounded device wait ran out left its output unspecified; the
// kernel posted that to the device's pending-error word, which is checked
// (without synchronising) before every launch, so the caller gets a
// RuntimeError here instead of using that output silently.  The word is
// cleared, so the call after this one runs normally.  Needs the operands'
// device current.
void check_pending() {
    uint32_t flags = 0;
    const int st = tinym_pending_errors(&flags, 1);
    TORCH_CHECK(st == TINYM_OK || st == TINYM_ERR_DEVICE_TIMEOUT, tinym_status_string(st), ": ",
                tinym_last_error());
    TORCH_CHECK(flags == 0u, "TINYM_ERR_DEVICE_TIMEOUT: ", tinym_last_error());
}

at::Tensor launch(const at::Tensor& a, const at::Tensor& b, const float* alpha_dev, float alpha) {
    const int64_t m = a.size(0), k = a.size(1), n = b.size(0);
    const c10::cuda::CUDAGuard guard(a.device());
    check_pending();
    at::Tensor y = at::empty({m, n}, a.options().dtype(at::ScalarType::BFloat16));
    if (m == 0 || n == 0) return y;
    cudaStream_t stream = at::cuda::getCurrentCUDAStream(a.get_device());
    const int st = tinym_fp8_gemm_ex(a.data_ptr(), b.data_ptr(), y.data_ptr(), n, m, n, k,
                                     alpha_dev, alpha, nullptr, stream);
    raise_status(st);
    return y;
}

at::Tensor run_host_alpha(const at::Tensor& a, const at::Tensor& b, double alpha) {
    check_inputs(a, b);
    TORCH_CHECK(std::isfinite(alpha), "alpha must be finite");
    return launch(a, b, nullptr, static_cast<float>(alpha));
}

at::Tensor run_alpha_tensor(const at::Tensor& a, const at::Tensor& b, const at::Tensor& alpha) {
    check_inputs(a, b);
    TORCH_CHECK(alpha.is_cuda() && alpha.scalar_type() == at::ScalarType::Float &&
                    alpha.numel() == 1,
                "alpha must be a one-element CUDA float32 tensor");
    TORCH_CHECK(alpha.get_device() == a.get_device(), "alpha must be on A's device");
    return launch(a, b, alpha.data_ptr<float>(), 0.0f);
}

at::Tensor pack_weights(const at::Tensor& b) {
    TORCH_CHECK(b.is_cuda(), "B must be a CUDA tensor");
    TORCH_CHECK(b.dim() == 2 && b.is_contiguous(), "B must be a contiguous rank-2 tensor");
    TORCH_CHECK(b.scalar_type() == at::ScalarType::Float8_e4m3fn,
                "B must have dtype torch.float8_e4m3fn");
    const int64_t n = b.size(0), k = b.size(1);
    int64_t bytes = 0;
    raise_status(tinym_packed_weight_bytes(n, k, &bytes));
    const c10::cuda::CUDAGuard guard(b.device());
    at::Tensor out = at::empty({bytes}, b.options().dtype(at::ScalarType::Byte));
    raise_status(tinym_pack_weights(b.data_ptr(), out.data_ptr(), n, k,
                                    at::cuda::getCurrentCUDAStream(b.get_device())));
    return out;
}

at::Tensor run_packed(const at::Tensor& a, const at::Tensor& bp, int64_t n, int64_t k,
                      const at::Tensor& alpha) {
    TORCH_CHECK(a.is_cuda() && bp.is_cuda(), "A and B must be CUDA tensors");
    TORCH_CHECK(a.get_device() == bp.get_device(), "A and B must be on the same CUDA device");
    TORCH_CHECK(a.dim() == 2 && a.is_contiguous(), "A must be a contiguous rank-2 tensor");
    TORCH_CHECK(a.scalar_type() == at::ScalarType::Float8_e4m3fn,
                "A must have dtype torch.float8_e4m3fn");
    TORCH_CHECK(a.size(1) == k, "A and B must have the same K dimension");
    TORCH_CHECK(bp.scalar_type() == at::ScalarType::Byte && bp.dim() == 1 && bp.is_contiguous(),
                "B_packed must be the uint8 tensor returned by pack_weights");
    int64_t bytes = 0;
    raise_status(tinym_packed_weight_bytes(n, k, &bytes));
    TORCH_CHECK(bp.numel() == bytes, "B_packed has ", num(bp.numel()), " bytes, packed [", num(n),
                ", ", num(k), "] needs ", num(bytes));
    TORCH_CHECK(alpha.is_cuda() && alpha.scalar_type() == at::ScalarType::Float &&
                    alpha.numel() == 1,
                "alpha must be a one-element CUDA float32 tensor");
    TORCH_CHECK(alpha.get_device() == a.get_device(), "alpha must be on A's device");
    const int64_t m = a.size(0);
    const c10::cuda::CUDAGuard guard(a.device());
    check_pending();
    at::Tensor y = at::empty({m, n}, a.options().dtype(at::ScalarType::BFloat16));
    if (m == 0 || n == 0) return y;
    raise_status(tinym_fp8_gemm_packed(a.data_ptr(), bp.data_ptr(), y.data_ptr(), n, m, n, k,
                                       alpha.data_ptr<float>(), 0.0f, nullptr,
                                       at::cuda::getCurrentCUDAStream(a.get_device())));
    return y;
}

std::tuple<at::Tensor, at::Tensor> run_quant_act(const at::Tensor& x, const at::Tensor& b,
                                                 const at::Tensor& w_scale) {
    TORCH_CHECK(x.is_cuda() && b.is_cuda() && w_scale.is_cuda(), "X, B and w_scale must be CUDA tensors");
    TORCH_CHECK(x.get_device() == b.get_device() && w_scale.get_device() == b.get_device(),
                "X, B and w_scale must be on the same CUDA device");
    TORCH_CHECK(x.dim() == 2 && b.dim() == 2, "X and B must both be rank-2 tensors");
    TORCH_CHECK(x.is_contiguous() && b.is_contiguous(), "X and B must be contiguous row-major tensors");
    TORCH_CHECK(x.scalar_type() == at::ScalarType::BFloat16 || x.scalar_type() == at::ScalarType::Float,
                "X must have dtype torch.bfloat16 or torch.float32");
    TORCH_CHECK(b.scalar_type() == at::ScalarType::Float8_e4m3fn, "B must have dtype torch.float8_e4m3fn");
    TORCH_CHECK(x.size(1) == b.size(1), "X and B must have the same K dimension");
    TORCH_CHECK(w_scale.scalar_type() == at::ScalarType::Float && w_scale.numel() == 1,
                "w_scale must be a one-element float32 tensor");
    const int64_t m = x.size(0), k = x.size(1), n = b.size(0);
    const c10::cuda::CUDAGuard guard(x.device());
    check_pending();
    at::Tensor y = at::empty({m, n}, b.options().dtype(at::ScalarType::BFloat16));
    int64_t ws_bytes = 0;
    raise_status(tinym_quant_workspace_bytes(m, k, &ws_bytes));
    at::Tensor ws = at::empty({ws_bytes}, b.options().dtype(at::ScalarType::Byte));
    const int dt = x.scalar_type() == at::ScalarType::BFloat16 ? TINYM_ACT_BF16 : TINYM_ACT_F32;
    raise_status(tinym_fp8_gemm_quant_act(x.data_ptr(), dt, b.data_ptr(), w_scale.data_ptr<float>(),
                                          y.data_ptr(), n, m, n, k, ws.data_ptr(), nullptr,
                                          at::cuda::getCurrentCUDAStream(x.get_device())));
    // x_scale is the workspace's first float (a view keeps the workspace alive).
    return {y, ws.narrow(0, 0, 4).view(at::ScalarType::Float)};
}

// ---------------------------------------------------------------- grouped and MXFP4 operators
void check_out(const at::Tensor& out, int64_t rows, int64_t n, const at::Tensor& a) {
    TORCH_CHECK(out.is_cuda() && out.get_device() == a.get_device(), "out must be on A's device");
    TORCH_CHECK(out.scalar_type() == at::ScalarType::BFloat16 && out.dim() == 2 &&
                    out.size(0) == rows && out.size(1) == n &&
                    (n == 1 || out.stride(1) == 1) && (rows <= 1 || out.stride(0) >= n),
                "out must be a [", num(rows), ", ", num(n), "] bfloat16 tensor with unit column stride");
}

int64_t out_stride(const at::Tensor& out) {  // one row: its stride says nothing
    return out.size(0) > 1 ? out.stride(0) : out.size(1);
}

// 0 (no alpha), 1 or `experts` values.
int check_alpha(const std::optional<at::Tensor>& alpha, int64_t experts, const at::Tensor& a) {
    if (!alpha.has_value()) return 0;
    TORCH_CHECK(alpha->is_cuda() && alpha->get_device() == a.get_device(), "alpha must be on A's device");
    TORCH_CHECK(alpha->scalar_type() == at::ScalarType::Float && alpha->is_contiguous() &&
                    (alpha->numel() == 1 || alpha->numel() == experts),
                "alpha must be a contiguous float32 tensor of 1 or ", num(experts), " values");
    return static_cast<int>(alpha->numel());
}

void check_offsets(const at::Tensor& offsets, int64_t experts, const at::Tensor& a) {
    TORCH_CHECK(offsets.is_cuda() && offsets.get_device() == a.get_device(),
                "offsets must be on A's device");
    TORCH_CHECK(offsets.scalar_type() == at::ScalarType::Int && offsets.dim() == 1 &&
                    offsets.is_contiguous() && offsets.numel() == experts + 1,
                "offsets must be a contiguous int32 vector of experts + 1 = ", num(experts + 1),
                " values");
}

// out undefined: a fresh Y, whose rows of no group are zeros.
at::Tensor grouped(const at::Tensor& a, const at::Tensor& b, const std::optional<at::Tensor>& alpha,
                   const at::Tensor& offsets, at::Tensor out) {
    TORCH_CHECK(a.is_cuda() && b.is_cuda(), "A and B must be CUDA tensors");
    TORCH_CHECK(a.get_device() == b.get_device(), "A and B must be on the same CUDA device");
    TORCH_CHECK(a.dim() == 2 && b.dim() == 3, "A must be [rows, K] and B [experts, N, K]");
    TORCH_CHECK(a.is_contiguous() && b.is_contiguous(), "A and B must be contiguous row-major tensors");
    TORCH_CHECK(a.scalar_type() == at::ScalarType::Float8_e4m3fn &&
                    b.scalar_type() == at::ScalarType::Float8_e4m3fn,
                "A and B must have dtype torch.float8_e4m3fn");
    TORCH_CHECK(a.size(1) == b.size(2), "A and B must have the same K dimension");
    const int64_t rows = a.size(0), k = a.size(1), experts = b.size(0), n = b.size(1);
    TORCH_CHECK(experts >= 1, "B must hold at least one expert");
    const int count = check_alpha(alpha, experts, a);
    check_offsets(offsets, experts, a);
    const c10::cuda::CUDAGuard guard(a.device());
    check_pending();
    const bool fresh = !out.defined();
    if (fresh) out = at::empty({rows, n}, a.options().dtype(at::ScalarType::BFloat16));
    else check_out(out, rows, n, a);
    if (rows == 0 || n == 0) return out;
    raise_status(tinym_fp8_gemm_grouped(a.data_ptr(), b.data_ptr(), out.data_ptr(), out_stride(out),
                                        rows, experts, n, k, offsets.data_ptr<int32_t>(),
                                        count ? alpha->data_ptr<float>() : nullptr, count,
                                        fresh ? TINYM_FLAG_ZERO_REST : 0u,
                                        at::cuda::getCurrentCUDAStream(a.get_device())));
    return out;
}

at::Tensor run_grouped(const at::Tensor& a, const at::Tensor& b, const at::Tensor& alpha,
                       const at::Tensor& offsets) {
    return grouped(a, b, alpha, offsets, at::Tensor());
}
void run_grouped_out(const at::Tensor& a, const at::Tensor& b, const at::Tensor& alpha,
                     const at::Tensor& offsets, at::Tensor out) {
    TORCH_CHECK(out.defined(), "out must be a tensor");
    grouped(a, b, alpha, offsets, out);
}

// Batch, rows and K of MXFP4 codes [.., rows, K / 2] with their scales.
struct MxShape {
    int64_t batch, rows, k;
};
MxShape check_mxfp4(const at::Tensor& codes, const at::Tensor& scales, const char* name) {
    TORCH_CHECK(codes.is_cuda() && scales.is_cuda() && codes.get_device() == scales.get_device(), name,
                " and its scales must be CUDA tensors on the same device");
    TORCH_CHECK(codes.scalar_type() == at::ScalarType::Byte && scales.scalar_type() == at::ScalarType::Byte,
                name, " and its scales must have dtype torch.uint8");
    TORCH_CHECK((codes.dim() == 2 || codes.dim() == 3) && codes.is_contiguous() && scales.is_contiguous(),
                name, " must be contiguous [rows, K / 2] or [batch, rows, K / 2] codes with contiguous scales");
    const int64_t d = codes.dim();
    const MxShape s{d == 3 ? codes.size(0) : 1, codes.size(d - 2), 2 * codes.size(d - 1)};
    TORCH_CHECK(s.k > 0 && s.k % 32 == 0, name, " must have K a positive multiple of 32 (got ", num(s.k), ")");
    const int64_t rb = (s.rows + 127) / 128, kb = (s.k + 127) / 128;
    TORCH_CHECK(scales.dim() == d + 1 && (d == 2 || scales.size(0) == s.batch) &&
                    scales.size(d - 2) == rb && scales.size(d - 1) == kb && scales.size(d) == 512,
                name, "'s scales must be [", (d == 3 ? "batch, " : ""), num(rb), ", ", num(kb),
                ", 512] as mxfp4_quantize lays them out");
    return s;
}

std::tuple<at::Tensor, at::Tensor> mxfp4_quantize(const at::Tensor& x) {
    TORCH_CHECK(x.is_cuda(), "X must be a CUDA tensor");
    TORCH_CHECK((x.dim() == 2 || x.dim() == 3) && x.is_contiguous(),
                "X must be a contiguous [rows, K] or [batch, rows, K] tensor");
    TORCH_CHECK(x.scalar_type() == at::ScalarType::BFloat16 || x.scalar_type() == at::ScalarType::Float,
                "X must have dtype torch.bfloat16 or torch.float32");
    const int64_t d = x.dim(), rows = x.size(d - 2), k = x.size(d - 1);
    TORCH_CHECK(k > 0 && k % 32 == 0, "X must have K a positive multiple of 32 (got ", num(k), ")");
    const int64_t batch = d == 3 ? x.size(0) : 1, rb = (rows + 127) / 128, kb = (k + 127) / 128;
    const c10::cuda::CUDAGuard guard(x.device());
    check_pending();
    const auto bytes = x.options().dtype(at::ScalarType::Byte);
    at::Tensor codes = d == 3 ? at::empty({batch, rows, k / 2}, bytes) : at::empty({rows, k / 2}, bytes);
    at::Tensor scales = d == 3 ? at::empty({batch, rb, kb, 512}, bytes) : at::empty({rb, kb, 512}, bytes);
    if (x.numel() == 0) return {codes, scales};
    const int dt = x.scalar_type() == at::ScalarType::BFloat16 ? TINYM_ACT_BF16 : TINYM_ACT_F32;
    raise_status(tinym_mxfp4_quantize(x.data_ptr(), dt, codes.data_ptr(), scales.data_ptr(), batch,
                                      rows, k, at::cuda::getCurrentCUDAStream(x.get_device())));
    return {codes, scales};
}

at::Tensor mxfp4_dequantize(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType dtype) {
    const MxShape s = check_mxfp4(codes, scales, "codes");
    TORCH_CHECK(dtype == at::ScalarType::BFloat16 || dtype == at::ScalarType::Float,
                "dtype must be torch.bfloat16 or torch.float32");
    const c10::cuda::CUDAGuard guard(codes.device());
    check_pending();
    const auto opt = codes.options().dtype(dtype);
    at::Tensor y = codes.dim() == 3 ? at::empty({s.batch, s.rows, s.k}, opt) : at::empty({s.rows, s.k}, opt);
    if (y.numel() == 0) return y;
    raise_status(tinym_mxfp4_dequantize(codes.data_ptr(), scales.data_ptr(), y.data_ptr(),
                                        dtype == at::ScalarType::BFloat16 ? TINYM_ACT_BF16 : TINYM_ACT_F32,
                                        s.batch, s.rows, s.k,
                                        at::cuda::getCurrentCUDAStream(codes.get_device())));
    return y;
}

// offsets undefined: the plain product (B [N, K / 2]).
at::Tensor mxfp4(const at::Tensor& a, const at::Tensor& as, const at::Tensor& b, const at::Tensor& bs,
                 const at::Tensor& offsets, const std::optional<at::Tensor>& alpha, at::Tensor out) {
    const MxShape sa = check_mxfp4(a, as, "A"), sb = check_mxfp4(b, bs, "B");
    TORCH_CHECK(a.get_device() == b.get_device(), "A and B must be on the same CUDA device");
    TORCH_CHECK(a.dim() == 2 && b.dim() == (offsets.defined() ? 3 : 2),
                offsets.defined() ? "A must be [rows, K / 2] and B [experts, N, K / 2]"
                                  : "A must be [M, K / 2] and B [N, K / 2]");
    TORCH_CHECK(sa.k == sb.k, "A and B must have the same K dimension");
    TORCH_CHECK(sb.batch >= 1, "B must hold at least one expert");
    const int count = check_alpha(alpha, sb.batch, a);
    if (offsets.defined()) check_offsets(offsets, sb.batch, a);
    const c10::cuda::CUDAGuard guard(a.device());
    check_pending();
    const bool fresh = !out.defined();
    if (fresh) out = at::empty({sa.rows, sb.rows}, a.options().dtype(at::ScalarType::BFloat16));
    else check_out(out, sa.rows, sb.rows, a);
    if (out.numel() == 0) return out;
    raise_status(tinym_mxfp4_gemm_grouped(
        a.data_ptr(), as.data_ptr(), b.data_ptr(), bs.data_ptr(), out.data_ptr(), out_stride(out),
        sa.rows, sb.batch, sb.rows, sa.k, offsets.defined() ? offsets.data_ptr<int32_t>() : nullptr,
        count ? alpha->data_ptr<float>() : nullptr, count, fresh ? TINYM_FLAG_ZERO_REST : 0u,
        at::cuda::getCurrentCUDAStream(a.get_device())));
    return out;
}

at::Tensor run_mxfp4(const at::Tensor& a, const at::Tensor& as, const at::Tensor& b,
                     const at::Tensor& bs, const std::optional<at::Tensor>& alpha) {
    return mxfp4(a, as, b, bs, at::Tensor(), alpha, at::Tensor());
}
void run_mxfp4_out(const at::Tensor& a, const at::Tensor& as, const at::Tensor& b,
                   const at::Tensor& bs, const std::optional<at::Tensor>& alpha, at::Tensor out) {
    TORCH_CHECK(out.defined(), "out must be a tensor");
    mxfp4(a, as, b, bs, at::Tensor(), alpha, out);
}
at::Tensor run_mxfp4_grouped(const at::Tensor& a, const at::Tensor& as, const at::Tensor& b,
                             const at::Tensor& bs, const at::Tensor& offsets,
                             const std::optional<at::Tensor>& alpha) {
    TORCH_CHECK(offsets.defined(), "offsets must be a tensor");
    return mxfp4(a, as, b, bs, offsets, alpha, at::Tensor());
}
void run_mxfp4_grouped_out(const at::Tensor& a, const at::Tensor& as, const at::Tensor& b,
                           const at::Tensor& bs, const at::Tensor& offsets,
                           const std::optional<at::Tensor>& alpha, at::Tensor out) {
    TORCH_CHECK(offsets.defined() && out.defined(), "offsets and out must be tensors");
    mxfp4(a, as, b, bs, offsets, alpha, out);
}

}  // namespace

TORCH_LIBRARY(sm120_fp8_gemm, module) {
    module.def("run(Tensor a, Tensor b, float alpha) -> Tensor");
    module.def("run_alpha_tensor(Tensor a, Tensor b, Tensor alpha) -> Tensor");
    module.def("pack_weights(Tensor b) -> Tensor");
    module.def("run_packed(Tensor a, Tensor b_packed, int n, int k, Tensor alpha) -> Tensor");
    module.def("run_quant_act(Tensor x, Tensor b, Tensor w_scale) -> (Tensor, Tensor)");
    module.def("run_grouped(Tensor a, Tensor b, Tensor alpha, Tensor offsets) -> Tensor");
    module.def("run_grouped_out(Tensor a, Tensor b, Tensor alpha, Tensor offsets, Tensor(a!) out) -> ()");
    module.def("mxfp4_quantize(Tensor x) -> (Tensor, Tensor)");
    module.def("mxfp4_dequantize(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
    module.def("run_mxfp4(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, Tensor? alpha=None) -> Tensor");
    module.def(
        "run_mxfp4_out(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, Tensor? alpha, Tensor(a!) out) -> ()");
    module.def(
        "run_mxfp4_grouped(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, Tensor offsets, "
        "Tensor? alpha=None) -> Tensor");
    module.def(
        "run_mxfp4_grouped_out(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, Tensor offsets, "
        "Tensor? alpha, Tensor(a!) out) -> ()");
}

TORCH_LIBRARY_IMPL(sm120_fp8_gemm, CUDA, module) {
    module.impl("run", &run_host_alpha);
    module.impl("run_alpha_tensor", &run_alpha_tensor);
    module.impl("pack_weights", &pack_weights);
    module.impl("run_packed", &run_packed);
    module.impl("run_quant_act", &run_quant_act);
    module.impl("run_grouped", &run_grouped);
    module.impl("run_grouped_out", &run_grouped_out);
    module.impl("mxfp4_quantize", &mxfp4_quantize);
    module.impl("mxfp4_dequantize", &mxfp4_dequantize);
    module.impl("run_mxfp4", &run_mxfp4);
    module.impl("run_mxfp4_out", &run_mxfp4_out);
    module.impl("run_mxfp4_grouped", &run_mxfp4_grouped);
    module.impl("run_mxfp4_grouped_out", &run_mxfp4_grouped_out);
}
