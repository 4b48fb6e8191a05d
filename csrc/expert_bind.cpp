// Python bindings of the FP8 products, the experts' bf16 product with its
// gradients, and SwiGLU (kiwi_b200._C.ops).  A bad argument raises ValueError
// before anything is launched.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/extension.h>

#include <optional>
#include <string>

#include "kiwi/gemm/fp8_gemm.hpp"
#include "kiwi/gemm/grouped_linear.hpp"
#include "kiwi/ops/swiglu.hpp"

namespace py = pybind11;
using namespace kiwi;

namespace {

using OptTensor = std::optional<torch::Tensor>;

cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void require(bool ok, const std::string& what) {
    if (!ok) throw py::value_error(what);
}

bool aligned16(const torch::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

/// `t` itself where TMA can read its rows in place (unit column stride, 16-byte
/// base and row stride), a contiguous copy otherwise.
torch::Tensor tma_rows(const torch::Tensor& t) {
    const bool in_place = (t.stride(1) == 1 || t.size(1) == 1) && aligned16(t) &&
                          (t.size(0) == 1 || (t.stride(0) >= t.size(1) && t.stride(0) * t.element_size() % 16 == 0));
    return in_place ? t : t.clone(at::MemoryFormat::Contiguous);  // contiguous() would keep a bad base
}

int64_t row_stride(const torch::Tensor& t) { return t.size(0) == 1 ? t.size(1) : t.stride(0); }

void check_fp8_operand(const torch::Tensor& x, const torch::Tensor& s, int64_t scale_rows, const torch::Device& dev,
                       const char* what) {
    const std::string w(what);
    require(x.is_cuda() && x.device() == dev && s.device() == dev, w + " and its scales must be on one CUDA device");
    require(x.scalar_type() == torch::kFloat8_e4m3fn && x.dim() == 2, w + " must be float8_e4m3fn [rows, K]");
    require(x.size(1) >= 16 && x.size(1) % 16 == 0, "K must be a positive multiple of 16");
    require(x.size(1) <= INT32_MAX - 256, "K must be below 2^31 - 256");
    require(s.scalar_type() == torch::kFloat32 && s.dim() == 2 && s.size(0) == scale_rows &&
                s.size(1) == (x.size(1) + 127) / 128,
            w + "'s scales must be fp32 [" + std::to_string(scale_rows) + ", " +
                std::to_string((x.size(1) + 127) / 128) + "]");
}

void check_counts(const torch::Tensor& c, const torch::Device& dev) {
    require(c.device() == dev && c.scalar_type() == torch::kInt32 && c.dim() == 1 && c.is_contiguous(),
            "counts must be a contiguous int32 [groups] tensor on the rows' device");
    require(c.size(0) >= 1 && c.size(0) <= 1024, "1 to 1024 groups are supported");
}

void check_row_scale(const OptTensor& s, int64_t rows, const torch::Device& dev) {
    if (!s) return;
    require(s->device() == dev && s->scalar_type() == torch::kFloat32 && s->dim() == 1 && s->size(0) == rows &&
                s->is_contiguous(),
            "row_scale must be a contiguous fp32 [rows] tensor on the rows' device");
}

void check_out(const torch::Tensor& out, int64_t rows, int64_t cols, torch::ScalarType type, const torch::Device& dev) {
    require(out.device() == dev && out.scalar_type() == type && out.dim() == 2 && out.size(0) == rows &&
                out.size(1) == cols && (cols == 1 || out.stride(1) == 1) && (rows == 1 || out.stride(0) >= cols),
            "out must be [" + std::to_string(rows) + ", " + std::to_string(cols) + "] with unit column stride, of the "
            "result's type, on the rows' device");
    require(!out.requires_grad() || !torch::GradMode::is_enabled(),
            "out requires a gradient: it can only be written under torch.no_grad()");
}

/// `out` was written: what saved it for a backward pass must find that out.
void written(const torch::Tensor& out) {
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}

/// Whether two tensors' storage ranges meet (an output must not be an input).
bool overlap(const torch::Tensor& x, const torch::Tensor& y) {
    auto range = [](const torch::Tensor& t) {
        const auto* b = static_cast<const char*>(t.data_ptr());
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
        return std::make_pair(b, b + (last + 1) * t.element_size());
    };
    if (x.numel() == 0 || y.numel() == 0) return false;
    const auto [x0, x1] = range(x);
    const auto [y0, y1] = range(y);
    return x0 < y1 && y0 < x1;
}

uint32_t* error_word(const torch::Tensor& t, const torch::Device& dev) {
    require(t.device() == dev && t.scalar_type() == torch::kInt32 && t.numel() == 1,
            "error must be an int32 tensor of one element on the rows' device");
    return reinterpret_cast<uint32_t*>(t.data_ptr<int32_t>());
}

struct Fp8Call {
    torch::Tensor a, a_scale, b, b_scale;  // kept alive until the launch
    gemm::Fp8GemmArgs args{};
};

/// Checked operands of a product over `groups` groups (0: dense).
Fp8Call fp8_call(const torch::Tensor& a, const torch::Tensor& a_scale, const torch::Tensor& b,
                 const torch::Tensor& b_scale, const OptTensor& counts) {
    const auto dev = a.device();
    const int64_t groups = counts ? counts->numel() : 1;
    if (counts) check_counts(*counts, dev);
    require(b.dim() == 2 && b.size(0) >= 1 && b.size(0) % groups == 0, "B must be [groups * N, K]");
    const int64_t n = b.size(0) / groups;
    require(a.dim() == 2 && a.size(1) == b.size(1), "A and B must share K");
    require(!counts || n % 128 == 0, "a grouped product needs N to be a multiple of 128");
    check_fp8_operand(a, a_scale, a.size(0), dev, "A");
    check_fp8_operand(b, b_scale, groups * ((n + 127) / 128), dev, "B");
    require(a.size(0) < (int64_t{1} << 31) - 256 && b.size(0) < (int64_t{1} << 31) - 256, "fewer than 2^31 rows");
    Fp8Call c;
    c.a = tma_rows(a);
    c.b = tma_rows(b);
    c.a_scale = a_scale.stride(1) == 1 || a_scale.size(1) == 1 ? a_scale : a_scale.contiguous();
    c.b_scale = b_scale.contiguous();
    c.args.a = static_cast<const uint8_t*>(c.a.data_ptr());
    c.args.lda = row_stride(c.a);
    c.args.b = static_cast<const uint8_t*>(c.b.data_ptr());
    c.args.ldb = row_stride(c.b);
    c.args.a_scale = c.a_scale.data_ptr<float>();
    c.args.a_scale_stride = row_stride(c.a_scale);
    c.args.b_scale = c.b_scale.data_ptr<float>();
    c.args.counts = counts ? counts->data_ptr<int32_t>() : nullptr;
    c.args.num_groups = static_cast<int32_t>(groups);
    c.args.n = static_cast<int32_t>(n);
    c.args.k = static_cast<int32_t>(a.size(1));
    c.args.rows = a.size(0);
    return c;
}

torch::Tensor fp8_gemm_out(torch::Tensor a, torch::Tensor a_scale, torch::Tensor b, torch::Tensor b_scale,
                           OptTensor counts, OptTensor out, bool swiglu, OptTensor row_scale, bool follows,
                           uint32_t* error) {
    require(a.is_cuda(), "A must be a CUDA tensor");
    const c10::cuda::CUDAGuard guard(a.device());
    Fp8Call c = fp8_call(a, a_scale, b, b_scale, counts);
    require(!swiglu || c.args.n % 256 == 0, "SwiGLU needs N to be a multiple of 256");
    check_row_scale(row_scale, a.size(0), a.device());
    const int64_t cols = swiglu ? c.args.n / 2 : c.args.n;
    torch::Tensor o;
    if (out) {
        check_out(*out, a.size(0), cols, torch::kBFloat16, a.device());
        for (const auto& t : {a, a_scale, b, b_scale}) require(!overlap(*out, t), "out must not overlap an input");
        if (row_scale) require(!overlap(*out, *row_scale), "out must not overlap an input");
        if (counts) require(!overlap(*out, *counts), "out must not overlap an input");
        o = *out;
    } else {
        o = torch::empty({a.size(0), cols}, a.options().dtype(torch::kBFloat16));
    }
    c.args.c = reinterpret_cast<__nv_bfloat16*>(o.data_ptr());
    c.args.ldc = row_stride(o);
    c.args.row_scale = row_scale ? row_scale->data_ptr<float>() : nullptr;
    c.args.swiglu = swiglu;
    c.args.zero_tail = !out && counts;
    c.args.follows = follows;
    c.args.error = error;
    gemm::fp8_gemm(c.args, cur_stream());
    if (out) written(o);
    return o;
}

torch::Tensor fp8_gemm_py(torch::Tensor a, torch::Tensor a_scale, torch::Tensor b, torch::Tensor b_scale,
                          OptTensor counts, OptTensor out, bool swiglu, OptTensor row_scale) {
    return fp8_gemm_out(a, a_scale, b, b_scale, counts, out, swiglu, row_scale, false, nullptr);
}

/// The gate and up product with its SwiGLU rows quantised to FP8.
std::pair<torch::Tensor, torch::Tensor> fp8_swiglu_quant(const torch::Tensor& a, const torch::Tensor& a_scale,
                                                         const torch::Tensor& b, const torch::Tensor& b_scale,
                                                         const torch::Tensor& counts, bool zero_tail,
                                                         bool feeds_next, uint32_t* error) {
    Fp8Call c = fp8_call(a, a_scale, b, b_scale, counts);
    require(c.args.n % 256 == 0, "SwiGLU needs N to be a multiple of 256");
    torch::Tensor codes = torch::empty({a.size(0), c.args.n / 2}, a.options());
    torch::Tensor scales = torch::empty({a.size(0), c.args.n / 256}, a_scale.options());
    c.args.codes = static_cast<uint8_t*>(codes.data_ptr());
    c.args.scales = scales.data_ptr<float>();
    c.args.swiglu = true;
    c.args.zero_tail = zero_tail;
    c.args.feeds_next = feeds_next;
    c.args.error = error;
    gemm::fp8_gemm(c.args, cur_stream());
    return {codes, scales};
}

py::tuple fp8_swiglu_py(torch::Tensor a, torch::Tensor a_scale, torch::Tensor b, torch::Tensor b_scale,
                        torch::Tensor counts) {
    require(a.is_cuda(), "A must be a CUDA tensor");
    const c10::cuda::CUDAGuard guard(a.device());
    auto r = fp8_swiglu_quant(a, a_scale, b, b_scale, counts, true, false, nullptr);
    return py::make_tuple(r.first, r.second);
}

torch::Tensor expert_ffn_fp8_py(torch::Tensor x, torch::Tensor x_scale, torch::Tensor w13, torch::Tensor w13_scale,
                                torch::Tensor w2, torch::Tensor w2_scale, torch::Tensor counts, OptTensor row_scale,
                                OptTensor out, OptTensor error) {
    require(x.is_cuda() && x.dim() == 2, "x must be a CUDA tensor [rows, H]");
    const int64_t groups = counts.numel();
    require(groups >= 1 && w13.dim() == 2 && w2.dim() == 2 && w13.size(0) % (2 * groups) == 0 &&
                w2.size(0) == groups * x.size(1) && w2.size(1) == w13.size(0) / (2 * groups),
            "w13 must be [E * 2F, H] and w2 [E * H, F]");
    const c10::cuda::CUDAGuard guard(x.device());
    // The second product's arguments are refused before the first is launched.
    check_row_scale(row_scale, x.size(0), x.device());
    if (out) {
        check_out(*out, x.size(0), x.size(1), torch::kBFloat16, x.device());
        for (const auto& t : {x, x_scale, w13, w13_scale, w2, w2_scale, counts})
            require(!overlap(*out, t), "out must not overlap an input");
        if (row_scale) require(!overlap(*out, *row_scale), "out must not overlap an input");
    }
    require(w2.size(0) < (int64_t{1} << 31) - 256, "fewer than 2^31 rows");
    require(x.size(1) % 128 == 0, "H must be a multiple of 128");
    check_fp8_operand(w2, w2_scale, w2.size(0) / 128, x.device(), "w2");
    uint32_t* word = error ? error_word(*error, x.device()) : nullptr;
    auto h = fp8_swiglu_quant(x, x_scale, w13, w13_scale, counts, false, true, word);
    return fp8_gemm_out(h.first, h.second, w2, w2_scale, counts, out, false, row_scale, true, word);
}

py::tuple quant_fp8_weights_py(torch::Tensor w) {
    require(w.is_cuda() && w.scalar_type() == torch::kBFloat16 && w.dim() == 2, "w must be a bf16 [rows, K] CUDA tensor");
    const c10::cuda::CUDAGuard guard(w.device());
    if (w.size(1) != 1 && w.stride(1) != 1) w = w.contiguous();
    torch::Tensor codes = torch::empty({w.size(0), w.size(1)}, w.options().dtype(torch::kFloat8_e4m3fn));
    torch::Tensor scales =
        torch::empty({(w.size(0) + 127) / 128, (w.size(1) + 127) / 128}, w.options().dtype(torch::kFloat32));
    gemm::quant_fp8_blocks(reinterpret_cast<const __nv_bfloat16*>(w.data_ptr()), row_stride(w), w.size(0), w.size(1),
                           static_cast<uint8_t*>(codes.data_ptr()), scales.data_ptr<float>(), cur_stream());
    return py::make_tuple(codes, scales);
}

const __nv_bfloat16* bf16_ptr(const torch::Tensor& t) { return reinterpret_cast<const __nv_bfloat16*>(t.data_ptr()); }

void check_bf16_rows(const torch::Tensor& t, const torch::Device& dev, const char* what) {
    require(t.is_cuda() && t.device() == dev && t.scalar_type() == torch::kBFloat16 && t.dim() == 2,
            std::string(what) + " must be a bf16 [rows, columns] CUDA tensor on the operands' device");
}

/// Sizes common to the grouped product and its gradients: w (or dw) [groups * n, k].
gemm::GroupedLinearArgs linear_args(int64_t rows, int64_t n, int64_t k, const torch::Tensor& counts,
                                    const torch::Device& dev) {
    check_counts(counts, dev);
    require(n >= 64 && n % 64 == 0 && k >= 64 && k % 64 == 0, "N and K must be multiples of 64");
    require(k <= INT32_MAX - 256, "K must be below 2^31 - 256");
    require(rows < (int64_t{1} << 31) - 256 && counts.numel() * n < (int64_t{1} << 31) - 256, "fewer than 2^31 rows");
    gemm::GroupedLinearArgs a{};
    a.counts = counts.data_ptr<int32_t>();
    a.num_groups = static_cast<int32_t>(counts.numel());
    a.n = static_cast<int32_t>(n);
    a.k = static_cast<int32_t>(k);
    a.rows = rows;
    return a;
}

/// The result tensor: `out`, checked, or a new one.
torch::Tensor linear_out(const OptTensor& out, int64_t rows, int64_t cols, torch::ScalarType type,
                         const torch::Tensor& like, std::initializer_list<torch::Tensor> inputs) {
    if (!out) return torch::empty({rows, cols}, like.options().dtype(type));
    check_out(*out, rows, cols, type, like.device());
    require(aligned16(*out) && (rows == 1 || out->stride(0) * out->element_size() % 16 == 0),
            "out's rows must start on 16-byte boundaries");
    for (const auto& t : inputs) require(!overlap(*out, t), "out must not overlap an input");
    return *out;
}

torch::Tensor linear_forward_py(torch::Tensor x, torch::Tensor w, torch::Tensor counts, OptTensor out) {
    check_bf16_rows(x, x.device(), "x");
    check_bf16_rows(w, x.device(), "w");
    const c10::cuda::CUDAGuard guard(x.device());
    require(w.size(1) == x.size(1) && counts.numel() >= 1 && w.size(0) % counts.numel() == 0,
            "w must be [groups * N, K] with x's K");
    auto a = linear_args(x.size(0), w.size(0) / counts.numel(), x.size(1), counts, x.device());
    const torch::Tensor xr = tma_rows(x), wr = tma_rows(w);
    torch::Tensor o = linear_out(out, x.size(0), a.n, torch::kBFloat16, x, {x, w, counts});
    a.x = bf16_ptr(xr);
    a.ldx = row_stride(xr);
    a.w = bf16_ptr(wr);
    a.ldw = row_stride(wr);
    a.out = o.data_ptr();
    a.ldo = row_stride(o);
    a.zero_tail = !out;
    gemm::grouped_linear_forward(a, cur_stream());
    if (out) written(o);
    return o;
}

torch::Tensor linear_dgrad_py(torch::Tensor dy, torch::Tensor w, torch::Tensor counts, OptTensor out) {
    check_bf16_rows(dy, dy.device(), "dy");
    check_bf16_rows(w, dy.device(), "w");
    const c10::cuda::CUDAGuard guard(dy.device());
    require(counts.numel() >= 1 && w.size(0) == counts.numel() * dy.size(1), "w must be [groups * N, K] with dy's N");
    auto a = linear_args(dy.size(0), dy.size(1), w.size(1), counts, dy.device());
    const torch::Tensor dr = tma_rows(dy), wr = tma_rows(w);
    torch::Tensor o = linear_out(out, dy.size(0), a.k, torch::kBFloat16, dy, {dy, w, counts});
    a.dy = bf16_ptr(dr);
    a.lddy = row_stride(dr);
    a.w = bf16_ptr(wr);
    a.ldw = row_stride(wr);
    a.out = o.data_ptr();
    a.ldo = row_stride(o);
    a.zero_tail = !out;
    gemm::grouped_linear_dgrad(a, cur_stream());
    if (out) written(o);
    return o;
}

torch::Tensor linear_wgrad_py(torch::Tensor dy, torch::Tensor x, torch::Tensor counts, OptTensor out,
                              bool accumulate) {
    check_bf16_rows(dy, dy.device(), "dy");
    check_bf16_rows(x, dy.device(), "x");
    const c10::cuda::CUDAGuard guard(dy.device());
    require(dy.size(0) == x.size(0), "dy and x must have the same rows");
    require(out || !accumulate, "accumulate needs an out to add to");
    const auto type = out ? out->scalar_type() : torch::kBFloat16;
    require(type == torch::kBFloat16 || type == torch::kFloat32, "out must be bf16 or fp32");
    auto a = linear_args(dy.size(0), dy.size(1), x.size(1), counts, dy.device());
    const torch::Tensor dr = tma_rows(dy), xr = tma_rows(x);
    torch::Tensor o = linear_out(out, counts.numel() * a.n, a.k, type, dy, {dy, x, counts});
    a.dy = bf16_ptr(dr);
    a.lddy = row_stride(dr);
    a.x = bf16_ptr(xr);
    a.ldx = row_stride(xr);
    a.out = o.data_ptr();
    a.ldo = row_stride(o);
    a.out_fp32 = type == torch::kFloat32;
    a.accumulate = accumulate;
    gemm::grouped_linear_wgrad(a, cur_stream());
    if (out) written(o);
    return o;
}

void check_swiglu(const torch::Tensor& y, const OptTensor& row_scale) {
    check_bf16_rows(y, y.device(), "y");
    require(y.size(1) >= 256 && y.size(1) % 256 == 0, "y must have a multiple of 256 columns (128 gate, 128 up, ...)");
    require(y.size(1) <= INT32_MAX - 256, "y must have fewer than 2^31 - 256 columns");
    check_row_scale(row_scale, y.size(0), y.device());
}

torch::Tensor swiglu_py(torch::Tensor y, OptTensor row_scale) {
    check_swiglu(y, row_scale);
    const c10::cuda::CUDAGuard guard(y.device());
    const torch::Tensor yr = tma_rows(y);
    torch::Tensor h = torch::empty({y.size(0), y.size(1) / 2}, y.options());
    ops::swiglu_forward(bf16_ptr(yr), row_stride(yr), row_scale ? row_scale->data_ptr<float>() : nullptr,
                        reinterpret_cast<__nv_bfloat16*>(h.data_ptr()), y.size(0), static_cast<int>(h.size(1)),
                        cur_stream());
    return h;
}

std::pair<torch::Tensor, OptTensor> swiglu_grad(torch::Tensor dh, torch::Tensor y, OptTensor row_scale,
                                                bool need_scale_grad) {
    check_swiglu(y, row_scale);
    check_bf16_rows(dh, y.device(), "dh");
    require(dh.size(0) == y.size(0) && dh.size(1) * 2 == y.size(1), "dh must be [rows, F] for y [rows, 2F]");
    require(row_scale || !need_scale_grad, "without row_scale there is no gradient of it");
    const c10::cuda::CUDAGuard guard(y.device());
    const torch::Tensor yr = tma_rows(y), dr = tma_rows(dh);
    torch::Tensor dy = torch::empty({y.size(0), y.size(1)}, y.options());
    OptTensor ds;
    if (need_scale_grad) ds = torch::empty({y.size(0)}, y.options().dtype(torch::kFloat32));
    ops::swiglu_backward(bf16_ptr(dr), row_stride(dr), bf16_ptr(yr), row_stride(yr),
                         row_scale ? row_scale->data_ptr<float>() : nullptr,
                         reinterpret_cast<__nv_bfloat16*>(dy.data_ptr()), ds ? ds->data_ptr<float>() : nullptr,
                         y.size(0), static_cast<int>(dh.size(1)), cur_stream());
    return {dy, ds};
}

// ---- autograd (CUDA tensors; the CPU restatements have their own in Python) ----

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

/// Passes a gradient on, and refuses to be differentiated: the gradients of this
/// file are once differentiable.  Its other arguments are what the gradient was
/// computed from.
struct OnceDifferentiable : torch::autograd::Function<OnceDifferentiable> {
    static torch::Tensor forward(AutogradContext*, torch::Tensor grad, torch::Tensor, torch::Tensor, OptTensor) {
        return grad.view_as(grad);
    }
    static variable_list backward(AutogradContext*, variable_list) {
        TORCH_CHECK(false, "the gradients of grouped_linear and swiglu are once differentiable");
    }
    static torch::Tensor mark(const torch::Tensor& grad, const torch::Tensor& a, const torch::Tensor& b,
                              const OptTensor& c = std::nullopt) {
        return grad.defined() && torch::GradMode::is_enabled() ? apply(grad, a, b, c) : grad;
    }
};

struct GroupedLinear : torch::autograd::Function<GroupedLinear> {
    static torch::Tensor forward(AutogradContext* ctx, torch::Tensor x, torch::Tensor w, torch::Tensor counts) {
        ctx->save_for_backward({x, w, counts});
        at::AutoDispatchBelowADInplaceOrView below;
        return linear_forward_py(x, w, counts, std::nullopt);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const torch::Tensor &x = saved[0], &w = saved[1], &counts = saved[2], &dy = grads[0];
        torch::Tensor dx, dw;
        if (dy.defined()) {
            at::AutoDispatchBelowADInplaceOrView below;
            if (ctx->needs_input_grad(0)) dx = linear_dgrad_py(dy, w, counts, std::nullopt);
            if (ctx->needs_input_grad(1)) dw = linear_wgrad_py(dy, x, counts, std::nullopt, false);
        }
        return {OnceDifferentiable::mark(dx, dy, w), OnceDifferentiable::mark(dw, dy, x), torch::Tensor()};
    }
};

struct SwiGLU : torch::autograd::Function<SwiGLU> {
    static torch::Tensor forward(AutogradContext* ctx, torch::Tensor y, OptTensor row_scale) {
        ctx->save_for_backward({y, row_scale ? *row_scale : torch::Tensor()});
        at::AutoDispatchBelowADInplaceOrView below;
        return swiglu_py(y, row_scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const torch::Tensor &y = saved[0], &s = saved[1], &dh = grads[0];
        if (!dh.defined()) return {torch::Tensor(), torch::Tensor()};
        std::pair<torch::Tensor, OptTensor> r;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            r = swiglu_grad(dh, y, s.defined() ? OptTensor(s) : std::nullopt, s.defined() && ctx->needs_input_grad(1));
        }
        const OptTensor scale = s.defined() ? OptTensor(s) : std::nullopt;
        return {OnceDifferentiable::mark(r.first, dh, y, scale),
                r.second ? OnceDifferentiable::mark(*r.second, dh, y, scale) : torch::Tensor()};
    }
};

/// Reads and clears an error word, or a device's (waits for the current stream).
int64_t take_error(const torch::Device& dev, uint32_t* word) {
    py::gil_scoped_release nogil;  // what it waits for may be waiting for a callback in Python
    const c10::cuda::CUDAGuard guard(dev);
    const torch::Tensor bits = torch::empty({1}, torch::dtype(torch::kInt32).device(dev));
    gemm::take_error(word ? word : gemm::gemm_error_word(), reinterpret_cast<uint32_t*>(bits.data_ptr<int32_t>()), cur_stream());
    return bits.item<int32_t>();
}

}  // namespace

void register_expert_ops(py::module_& m) {
    py::module_ o = m.attr("ops").cast<py::module_>();
    o.def("fp8_gemm", &fp8_gemm_py, py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"),
          py::arg("counts") = py::none(), py::arg("out") = py::none(), py::arg("swiglu") = false,
          py::arg("row_scale") = py::none(),
          "Block-scaled FP8 product, dense or grouped by device row counts, bf16 out.  Current stream.");
    o.def("fp8_swiglu", &fp8_swiglu_py, py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"),
          py::arg("counts"), "Grouped FP8 product with SwiGLU, its rows quantised 1x128: (codes, scales).");
    o.def("expert_ffn_fp8", &expert_ffn_fp8_py, py::arg("x"), py::arg("x_scale"), py::arg("w13"), py::arg("w13_scale"),
          py::arg("w2"), py::arg("w2_scale"), py::arg("counts"), py::arg("row_scale") = py::none(),
          py::arg("out") = py::none(), py::arg("error") = py::none(),
          "The experts' SwiGLU FFN on FP8 rows and weights (two launches); errors go into `error` (int32 [1]) if given.");
    o.def("quant_fp8_weights", &quant_fp8_weights_py, py::arg("w"),
          "128x128 FP8 e4m3 quantisation of a bf16 matrix: (codes, fp32 scales).");
    o.def("grouped_linear", [](torch::Tensor x, torch::Tensor w, torch::Tensor counts) {
        return GroupedLinear::apply(x, w, counts);
    }, py::arg("x"), py::arg("w"), py::arg("counts"), "y = x . w[g]^T for each group's rows; differentiable.");
    o.def("grouped_linear_out", [](torch::Tensor x, torch::Tensor w, torch::Tensor counts, torch::Tensor out) {
        return linear_forward_py(x, w, counts, out);
    }, py::arg("x"), py::arg("w"), py::arg("counts"), py::arg("out"), "The same into out; not differentiable.");
    o.def("grouped_linear_dgrad", &linear_dgrad_py, py::arg("dy"), py::arg("w"), py::arg("counts"),
          py::arg("out") = py::none(), "dx = dy . w[g] for each group's rows.");
    o.def("grouped_linear_wgrad", &linear_wgrad_py, py::arg("dy"), py::arg("x"), py::arg("counts"),
          py::arg("out") = py::none(), py::arg("accumulate") = false, "dw[g] (+)= dy^T . x over each group's rows.");
    o.def("swiglu", [](torch::Tensor y, OptTensor row_scale) { return SwiGLU::apply(y, row_scale); }, py::arg("y"),
          py::arg("row_scale") = py::none(),
          "row_scale * silu(gate) * up of rows in blocks of 128 gate and 128 up columns; differentiable.");
    o.def("swiglu_grad", &swiglu_grad, py::arg("dh"), py::arg("y"), py::arg("row_scale") = py::none(),
          py::arg("need_scale_grad") = false, "(dy, drow_scale or None) of swiglu.");
    o.def("gemm_error", [](int64_t device) {
        return take_error(torch::Device(torch::kCUDA, static_cast<c10::DeviceIndex>(device)), nullptr);
    }, py::arg("device"), "Reads and clears the products' error word of a device.");
    o.def("take_error", [](const torch::Tensor& error) {
        require(error.is_cuda(), "error must be a CUDA tensor");
        return take_error(error.device(), error_word(error, error.device()));
    }, py::arg("error"), "Reads and clears an error word of its caller's own.");
}
