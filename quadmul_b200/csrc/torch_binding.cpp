// Compiled PyTorch binding of the entry points that are called per layer: module `_quadmul_torch`.
//
// gemm is the reference's extension function (extension.cpp:8-24, registered at extension.cpp:26-29):
// gemm(a, b, c, m, n, k) with packed A (m x k/2), packed B (n x k/2), int32 C (m x n), launched on the current
// stream of a's device, returning None.  Unlike the reference it checks its arguments, makes a's device current
// for the call, and raises when the library reports an error.  The others are the calls of w4.py and moe.py, with the same
// checks and the same errors as their ctypes forms.  Everything here only marshals: the work is in the library.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>

#include "../../include/quadmul_b200.h"

namespace py = pybind11;

namespace {

void check_operands(const torch::Tensor &a, const torch::Tensor &b, const torch::Tensor &c, int64_t m, int64_t n, int64_t k)
{
    TORCH_CHECK(a.is_cuda() && b.is_cuda() && c.is_cuda(), "quadmul.gemm: a, b and c must be CUDA tensors");
    TORCH_CHECK(a.device() == b.device() && a.device() == c.device(), "quadmul.gemm: a, b and c must be on the same device");
    TORCH_CHECK(c.scalar_type() == torch::kInt32, "quadmul.gemm: c must be int32");
    TORCH_CHECK(a.element_size() == 1 && b.element_size() == 1, "quadmul.gemm: a and b must be 1-byte tensors (two nibbles per byte)");
    TORCH_CHECK(a.is_contiguous() && b.is_contiguous() && c.is_contiguous(), "quadmul.gemm: tensors must be contiguous");
    TORCH_CHECK(m >= 0 && n >= 0 && k >= 0 && m <= INT32_MAX && n <= INT32_MAX && k <= INT32_MAX, "quadmul.gemm: bad m, n, k");
    TORCH_CHECK(a.numel() >= m * (k / 2) && b.numel() >= n * (k / 2) && c.numel() >= m * n,
                "quadmul.gemm: tensor smaller than m, n, k imply");
}

void gemm(torch::Tensor a, torch::Tensor b, torch::Tensor c, int64_t m, int64_t n, int64_t k)
{
    check_operands(a, b, c, m, n, k);
    c10::cuda::CUDAGuard guard(a.device());
    const int st = qm_gemm_s4(a.data_ptr(), b.data_ptr(), c.data_ptr(), (int)m, (int)n, (int)k,
                              at::cuda::getCurrentCUDAStream(a.get_device()).stream());
    TORCH_CHECK(st == QM_OK, "quadmul.gemm(m=", m, ", n=", n, ", k=", k, "): ", qm_status_string(st), " ", qm_last_cuda_error());
}

// Kernels that the calls below have launched (the interpreter's lock is held: they run one at a time)
int64_t launched = 0;

using at::Tensor;
using OptTensor = std::optional<Tensor>;

[[noreturn]] void bad_value(const char *what, const std::string &why) { throw py::value_error(std::string(what) + ": " + why); }
[[noreturn]] void bad_type(const char *what, const std::string &why) { throw py::type_error(std::string(what) + ": " + why); }

int type_code(const char *what, const char *name, const Tensor &t)
{
    switch (t.scalar_type()) {
        case at::kFloat: return QM_TYPE_F32;
        case at::kHalf: return QM_TYPE_F16;
        case at::kBFloat16: return QM_TYPE_BF16;
        default: bad_type(what, std::string(name) + " is " + c10::toString(t.scalar_type()));
    }
}

void check_device(const char *what, const char *name, const Tensor &t, c10::Device device)
{
    if (!t.is_cuda() || t.device() != device) bad_value(what, std::string(name) + " must be a CUDA tensor on " + device.str());
    if (t.requires_grad() && at::GradMode::is_enabled()) bad_value(what, std::string(name) + " requires a gradient, which this call does not record");
}

// 2-D, rows contiguous and not overlapping
void check_rows(const char *what, const char *name, const Tensor &t, c10::Device device)
{
    if (!t.is_cuda()) bad_value(what, std::string(name) + " must be a CUDA tensor (there is no CPU path)");
    check_device(what, name, t, device);
    if (t.dim() != 2) bad_value(what, std::string(name) + " must have two dimensions");
    if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)))
        bad_value(what, std::string("the rows of ") + name + " must be contiguous and must not overlap");
    if (t.size(0) > INT32_MAX || t.size(1) > INT32_MAX) bad_value(what, std::string(name) + " is too large");
}

void check_whole(const char *what, const char *name, const Tensor &t, c10::Device device)
{
    check_device(what, name, t, device);
    if (!t.is_contiguous()) bad_value(what, std::string(name) + " must be contiguous");
}

int64_t pitch(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1); }

Tensor checked_out(const char *what, const OptTensor &out, int64_t rows, int64_t cols, const Tensor &like)
{
    if (!out) return at::empty({rows, cols}, like.options().requires_grad(false));
    if (out->scalar_type() != like.scalar_type()) bad_type(what, "out has another type than the input");
    if (out->dim() != 2 || out->size(0) != rows || out->size(1) != cols) bad_value(what, "out has another shape than the result");
    check_rows(what, "out", *out, like.device());
    return *out;
}

void *stream_of(const Tensor &t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

void check_status(const char *what, int st)
{
    if (st != QM_OK) throw std::runtime_error(std::string(what) + ": " + qm_status_string(st) + (st == QM_ERR_CUDA ? std::string(" [") + qm_last_cuda_error() + "]" : ""));
}

struct Weights {
    int type, scale_type;
    int64_t n, k;
};

Weights check_weights(const char *what, const Tensor &x, const Tensor &b, const Tensor &scales, int64_t group, bool experts)
{
    if (b.dim() != (experts ? 3 : 2)) bad_value(what, experts ? "b must be [experts, n, k/2]" : "b must be [n, k/2]");
    Weights w;
    w.type = type_code(what, "x", x);
    if (w.type == QM_TYPE_F32) bad_type(what, "x must be float16 or bfloat16");
    if (!x.is_cuda()) bad_value(what, "x must be a CUDA tensor (there is no CPU path)");
    check_rows(what, "x", x, x.device());
    check_whole(what, "b", b, x.device());
    check_whole(what, "scales", scales, x.device());
    if (b.scalar_type() != at::kChar && b.scalar_type() != at::kByte) bad_type(what, "b must be int8 or uint8, two codes per byte");
    w.scale_type = type_code(what, "scales", scales);
    if (w.scale_type != w.type && w.scale_type != QM_TYPE_F32) bad_type(what, "scales must have x's type or be float32");
    if (group != 32 && group != 64 && group != 128 && group != 256) bad_value(what, "group must be one of (32, 64, 128, 256)");
    w.k = x.size(1);
    if (w.k % 2) bad_value(what, "k must be even");
    const int64_t lead = experts ? 1 : 0;
    if (b.size(lead + 1) != w.k / 2) bad_value(what, "b and x differ in k");
    w.n = b.size(lead);
    if (w.n > INT32_MAX) bad_value(what, "b is too large");
    if (scales.dim() != lead + 2 || (experts && scales.size(0) != b.size(0)) || scales.size(lead) != w.n || scales.size(lead + 1) != (w.k + group - 1) / group)
        bad_value(what, "scales must be [..., n, ceil(k / group)]");
    return w;
}

// the copies of operands that the kernels cannot address as they are (empty: none are needed)
Tensor workspace_for(const Tensor &x, const Tensor &b, int64_t experts, const Weights &w)
{
    const size_t need = qm_gemm_w4_workspace_bytes(x.data_ptr(), pitch(x), b.data_ptr(), (int)experts, (int)x.size(0), (int)w.n, (int)w.k);
    return need ? at::empty({(int64_t)need}, x.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}

// The product's kernel and the copies in front of it
int64_t product_launches(const Tensor &x, const Tensor &b, int64_t experts, const Weights &w)
{
    if (x.size(0) == 0 || w.n == 0 || experts == 0) return 0;
    if (w.k == 0) return 1;
    auto off = [&](const Tensor &t) { return w.k % 32 != 0 || (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) != 0; };
    return 1 + (off(x) || pitch(x) % 8 != 0) + off(b);
}

Tensor gemm_w4(const Tensor &x, const Tensor &b, const Tensor &scales, int64_t group, const OptTensor &out)
{
    const char *what = "gemm_w4";
    const Weights w = check_weights(what, x, b, scales, group, false);
    Tensor y = checked_out(what, out, x.size(0), w.n, x);
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor space = workspace_for(x, b, 1, w);
    check_status(what, qm_gemm_w4(x.data_ptr(), w.type, pitch(x), b.data_ptr(), scales.data_ptr(), w.scale_type, (int)group, y.data_ptr(), pitch(y),
                                  (int)x.size(0), (int)w.n, (int)w.k, space.defined() ? space.data_ptr() : nullptr,
                                  space.defined() ? space.numel() : 0, stream_of(x)));
    launched += product_launches(x, b, 1, w);
    return y;
}

Tensor moe_gemm_w4(const Tensor &x, const Tensor &b, const Tensor &scales, const Tensor &offsets, int64_t group, const OptTensor &out)
{
    const char *what = "moe_gemm_w4";
    const Weights w = check_weights(what, x, b, scales, group, true);
    check_whole(what, "offsets", offsets, x.device());
    if (offsets.scalar_type() != at::kInt || offsets.dim() != 1 || offsets.size(0) != b.size(0) + 1)
        bad_value(what, "offsets must be int32 of experts + 1 elements");
    if (b.size(0) > INT32_MAX) bad_value(what, "b is too large");
    Tensor y = checked_out(what, out, x.size(0), w.n, x);
    c10::cuda::CUDAGuard guard(x.device());
    const Tensor space = workspace_for(x, b, b.size(0), w);
    check_status(what, qm_moe_gemm_w4(x.data_ptr(), w.type, pitch(x), b.data_ptr(), scales.data_ptr(), w.scale_type, (int)group,
                                      static_cast<const int *>(offsets.data_ptr()), (int)b.size(0), y.data_ptr(), pitch(y), (int)x.size(0), (int)w.n,
                                      (int)w.k, space.defined() ? space.data_ptr() : nullptr, space.defined() ? space.numel() : 0, stream_of(x)));
    launched += product_launches(x, b, b.size(0), w);
    return y;
}

std::tuple<Tensor, Tensor> quantize_w4(const Tensor &w, int64_t group, bool float_scales)
{
    const char *what = "quantize_w4";
    const int type = type_code(what, "w", w);
    if (!w.is_cuda()) bad_value(what, "w must be a CUDA tensor (there is no CPU path)");
    check_rows(what, "w", w, w.device());
    if (group != 32 && group != 64 && group != 128 && group != 256) bad_value(what, "group must be one of (32, 64, 128, 256)");
    const int64_t n = w.size(0), k = w.size(1);
    if (k % 2) bad_value(what, "k must be even");
    Tensor packed = at::empty({n, k / 2}, w.options().dtype(at::kChar).requires_grad(false));
    Tensor scales = at::empty({n, (k + group - 1) / group}, w.options().dtype(float_scales ? at::kFloat : w.scalar_type()).requires_grad(false));
    c10::cuda::CUDAGuard guard(w.device());
    check_status(what, qm_quantize_w4(w.data_ptr(), type, pitch(w), packed.data_ptr(), scales.data_ptr(), float_scales ? QM_TYPE_F32 : type, n, k,
                                      (int)group, stream_of(w)));
    launched += n > 0 && k > 0;
    return {packed, scales};
}

std::tuple<Tensor, Tensor, Tensor> moe_sort(const Tensor &x, const Tensor &ids, int64_t experts, const OptTensor &out)
{
    const char *what = "moe_sort";
    const int type = type_code(what, "x", x);
    if (!x.is_cuda()) bad_value(what, "x must be a CUDA tensor (there is no CPU path)");
    check_rows(what, "x", x, x.device());
    check_whole(what, "expert_ids", ids, x.device());
    if (ids.dim() != 2 || ids.size(0) != x.size(0)) bad_value(what, "expert_ids must be [tokens, top_k]");
    if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) bad_type(what, "expert_ids must be int32 or int64");
    if (experts < 0 || experts > 4096) bad_value(what, "num_experts must be within [0, 4096]");
    const int64_t tokens = x.size(0), hidden = x.size(1), top_k = ids.size(1);
    if (top_k > 4096 || tokens * top_k > INT32_MAX) bad_value(what, "too many assignments");
    Tensor xs = checked_out(what, out, tokens * top_k, hidden, x);
    const auto ints = x.options().dtype(at::kInt).requires_grad(false);
    Tensor offsets = at::empty({experts + 1}, ints), slots = at::empty({tokens, top_k}, ints);
    const size_t need = qm_moe_sort_workspace_bytes((int)tokens, (int)top_k, (int)experts);
    Tensor workspace;
    if (need) workspace = at::empty({(int64_t)need / 4}, ints);
    c10::cuda::CUDAGuard guard(x.device());
    check_status(what, qm_moe_sort(x.data_ptr(), type, pitch(x), ids.data_ptr(), (int)ids.element_size(), (int)experts, xs.data_ptr(), pitch(xs),
                                   static_cast<int *>(offsets.data_ptr()), static_cast<int *>(slots.data_ptr()), (int)tokens, (int)top_k, (int)hidden,
                                   need ? workspace.data_ptr() : nullptr, need, stream_of(x)));
    launched += need ? 3 : 1;
    return {xs, offsets, slots};
}

void check_slots(const char *what, const Tensor &slots, c10::Device device)
{
    if (slots.dim() != 2 || slots.scalar_type() != at::kInt) bad_value(what, "slots must be int32 [tokens, top_k]");
    check_whole(what, "slots", slots, device);
    if (slots.size(0) > INT32_MAX || slots.size(1) > 4096 || slots.numel() > INT32_MAX) bad_value(what, "too many assignments");
}

int check_routing_weights(const char *what, const Tensor &weights, const Tensor &slots, const Tensor &like)
{
    check_whole(what, "weights", weights, like.device());
    if (weights.sizes() != slots.sizes()) bad_value(what, "weights and slots differ in shape");
    if (weights.scalar_type() != like.scalar_type() && weights.scalar_type() != at::kFloat) bad_type(what, "weights must have the rows' type or be float32");
    return type_code(what, "weights", weights);
}

Tensor moe_combine(const Tensor &ys, const Tensor &slots, const OptTensor &weights, const OptTensor &out)
{
    const char *what = "moe_combine";
    const int type = type_code(what, "ys", ys);
    if (!ys.is_cuda()) bad_value(what, "ys must be a CUDA tensor (there is no CPU path)");
    check_rows(what, "ys", ys, ys.device());
    check_slots(what, slots, ys.device());
    const int weight_type = weights ? check_routing_weights(what, *weights, slots, ys) : type;
    Tensor y = checked_out(what, out, slots.size(0), ys.size(1), ys);
    c10::cuda::CUDAGuard guard(ys.device());
    check_status(what, qm_moe_combine(ys.data_ptr(), type, pitch(ys), (int)ys.size(0), static_cast<const int *>(slots.data_ptr()),
                                      weights ? weights->data_ptr() : nullptr, weight_type, y.data_ptr(), pitch(y), (int)slots.size(0), (int)slots.size(1),
                                      (int)ys.size(1), stream_of(ys)));
    launched += y.numel() > 0;
    return y;
}

std::tuple<Tensor, Tensor> moe_combine_grad(const Tensor &dy, const Tensor &ys, const Tensor &slots, const Tensor &weights, const OptTensor &out)
{
    const char *what = "moe_combine_grad";
    const int type = type_code(what, "dy", dy);
    if (type_code(what, "ys", ys) != type) bad_type(what, "dy and ys differ in type");
    if (!dy.is_cuda()) bad_value(what, "dy must be a CUDA tensor (there is no CPU path)");
    check_rows(what, "dy", dy, dy.device());
    check_rows(what, "ys", ys, dy.device());
    check_slots(what, slots, ys.device());
    const int weight_type = check_routing_weights(what, weights, slots, ys);
    if (dy.size(0) != slots.size(0) || dy.size(1) != ys.size(1)) bad_value(what, "dy must be [tokens, hidden]");
    Tensor dys = checked_out(what, out, ys.size(0), ys.size(1), ys), dweights = at::empty(weights.sizes(), weights.options().requires_grad(false));
    c10::cuda::CUDAGuard guard(ys.device());
    check_status(what, qm_moe_combine_grad(dy.data_ptr(), pitch(dy), ys.data_ptr(), pitch(ys), type, (int)ys.size(0), static_cast<const int *>(slots.data_ptr()),
                                           weights.data_ptr(), weight_type, dys.data_ptr(), pitch(dys), dweights.data_ptr(), (int)slots.size(0),
                                           (int)slots.size(1), (int)ys.size(1), stream_of(ys)));
    launched += dweights.numel() > 0;
    return {dys, dweights};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod)
{
    mod.def("gemm", &gemm, "packed int4 x int4 -> int32 matrix product on B200 (C = A * B^T)");
    mod.def("gemm_w4", &gemm_w4, "16-bit x packed 4-bit weights with group scales");
    mod.def("moe_gemm_w4", &moe_gemm_w4, "gemm_w4 with one matrix per expert over sorted rows");
    mod.def("quantize_w4", &quantize_w4, "weights -> packed codes and group scales");
    mod.def("moe_sort", &moe_sort, "rows in expert order, offsets, slots");
    mod.def("moe_combine", &moe_combine, "weighted sum of the experts' rows per token");
    mod.def("moe_combine_grad", &moe_combine_grad, "gradients of moe_combine");
    mod.def("launched", [] { return launched; }, "kernels that the calls other than gemm have launched");
}
