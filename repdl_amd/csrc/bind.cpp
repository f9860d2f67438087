// repdl_amd.backend._hip_ext -- the compiled counterpart of RepDL's repdl.backend.cuda
// (backend/cuda/bind.cpp:6-19): a PyTorch C++ extension module that exports the same ten
// functions with the same positional signatures (matrix_multiplication.cu:234-235, 267;
// convolution.cu:153-155, 259-262, 359-362, 385-387; summation.cu:149-155;
// softmax.cpp:15, 28; cross_entropy.cpp:15, 31), plus exp / log / sqrt / div / div_scalar and
// mm_bias / conv2d_bias (the layer's bias added in the kernel's epilogue) and the fused elementwise
// passes of batch normalisation (bn_apply, bn_gvar_term, bn_gweight_term), layer normalisation, dropout and
// the preference loss with their gradients.
// It is the only file of this library that knows about PyTorch: every function checks its
// tensors, allocates the output on the input's device, and hands raw pointers and the current
// stream to the C ABI of include/repdl_hip.h.  Host C++ only; built with the host compiler
// against the PyTorch headers (repdl_amd/build.py, build_ext).
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "../../include/repdl_hip.h"

namespace repdl
{
namespace hip
{
namespace
{
// PyTorch-ROCm presents HIP devices and streams under the CUDA names.
using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;

void *current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

torch::Tensor checked(const torch::Tensor &t, const char *name, int64_t dim, c10::ScalarType dtype = torch::kFloat)
{
    TORCH_CHECK(t.is_cuda(), name, " must be on the GPU (this backend has no CPU path)");
    TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
    TORCH_CHECK(dim < 0 || t.dim() == dim, name, " must have ", dim, " dimensions, got ", t.dim());
    return t.contiguous();
}

void same_device(const torch::Tensor &a, const torch::Tensor &b)
{
    TORCH_CHECK(a.device() == b.device(), "tensors are on different devices: ", a.device(), " and ", b.device());
}

void ok(int rc, const char *what) { TORCH_CHECK(rc == 0, what, " failed with code ", rc, ": ", repdl_hip_error_string(rc)); }

// Scratch memory of a call from PyTorch's allocator (the *_ws entry points): the library then allocates,
// frees and keeps nothing of its own, and the call can be captured into a graph like any PyTorch operator.
// The tensor dies when the binding returns; PyTorch hands its memory to later work on the same stream only.
struct Scratch
{
    torch::Tensor hold;
    size_t bytes;
    Scratch(size_t nbytes, const torch::Tensor &like) : bytes(nbytes)
    {
        if (nbytes > 0)
            hold = torch::empty({(int64_t)nbytes}, like.options().dtype(torch::kUInt8));
    }
    void *ptr() const { return bytes > 0 ? hold.data_ptr() : nullptr; }
};
} // namespace

namespace
{
// the bias of a layer: [channels] on the same device, or none
const float *bias_pointer(const c10::optional<torch::Tensor> &bias, torch::Tensor &hold, const torch::Tensor &like,
                          int64_t channels)
{
    if (!bias.has_value())
        return nullptr;
    hold = checked(*bias, "bias", 1);
    same_device(hold, like);
    TORCH_CHECK(hold.size(0) == channels, "bias has ", hold.size(0), " elements for ", channels, " output channels");
    return hold.data_ptr<float>();
}
} // namespace

// mm followed by `+= bias` (repdl/nn/linear.py:21-22) with the addition in the kernel's epilogue
torch::Tensor mm_bias(const torch::Tensor &input, const torch::Tensor &mat2, const c10::optional<torch::Tensor> &bias,
                      bool transA, bool transB)
{
    const auto a = checked(input, "input", 2), b = checked(mat2, "mat2", 2);
    same_device(a, b);
    const int64_t M = !transA ? a.size(0) : a.size(1), K = !transA ? a.size(1) : a.size(0);
    const int64_t N = !transB ? b.size(1) : b.size(0), Kb = !transB ? b.size(0) : b.size(1);
    TORCH_CHECK(K == Kb, "mm: inner dimensions differ (", K, " vs ", Kb, ")");
    const DeviceGuard guard(a.device());
    torch::Tensor hold;
    const float *bp = bias_pointer(bias, hold, a, N);
    auto out = torch::empty({M, N}, a.options());
    ok(repdl_hip_mm_bias(a.data_ptr<float>(), b.data_ptr<float>(), bp, out.data_ptr<float>(), M, N, K, transA, transB,
                         current_stream()),
       "repdl_hip_mm");
    return out;
}

torch::Tensor mm(const torch::Tensor &input, const torch::Tensor &mat2, bool transA, bool transB)
{
    return mm_bias(input, mat2, c10::nullopt, transA, transB);
}

// conv2d followed by `+= bias` per output channel (repdl/nn/conv.py:27-28), the addition in the epilogue
torch::Tensor conv2d_bias(const torch::Tensor &input, const torch::Tensor &kernel, const c10::optional<torch::Tensor> &bias,
                          int64_t sH, int64_t sW, int64_t pH, int64_t pW, int64_t groups)
{
    const auto x = checked(input, "input", 4), k = checked(kernel, "kernel", 4);
    same_device(x, k);
    const int64_t N = x.size(0), IC = x.size(1), H = x.size(2), W = x.size(3);
    const int64_t OC = k.size(0), ICg = k.size(1), KH = k.size(2), KW = k.size(3);
    TORCH_CHECK(groups > 0 && IC % groups == 0 && OC % groups == 0 && ICg == IC / groups, "conv2d: channels (", IC,
                " in, ", OC, " out, kernel ", ICg, ") do not match groups=", groups);
    TORCH_CHECK(sH > 0 && sW > 0 && pH >= 0 && pW >= 0, "conv2d: bad stride or padding");
    TORCH_CHECK(H + 2 * pH >= KH && W + 2 * pW >= KW, "conv2d: kernel larger than padded input");
    const int64_t OH = (H + 2 * pH - KH) / sH + 1, OW = (W + 2 * pW - KW) / sW + 1;
    const DeviceGuard guard(x.device());
    torch::Tensor hold;
    const float *bp = bias_pointer(bias, hold, x, OC);
    auto out = torch::empty({N, OC, OH, OW}, x.options());
    const Scratch work(repdl_hip_conv2d_workspace_bytes(x.data_ptr<float>(), k.data_ptr<float>(), N, IC, H, W, OC, KH, KW, sH, sW,
                                                        pH, pW, groups),
                       x);
    ok(repdl_hip_conv2d_ws(x.data_ptr<float>(), k.data_ptr<float>(), bp, out.data_ptr<float>(), N, IC, H, W, OC, KH, KW, sH,
                           sW, pH, pW, groups, work.ptr(), work.bytes, current_stream()),
       "repdl_hip_conv2d_ws");
    return out;
}

torch::Tensor conv2d(const torch::Tensor &input, const torch::Tensor &kernel, int64_t sH, int64_t sW, int64_t pH,
                     int64_t pW, int64_t groups)
{
    return conv2d_bias(input, kernel, c10::nullopt, sH, sW, pH, pW, groups);
}

torch::Tensor conv2d_grad_input(const torch::Tensor &grad_output, const torch::Tensor &kernel, int64_t H, int64_t W,
                                int64_t sH, int64_t sW, int64_t pH, int64_t pW)
{
    const auto go = checked(grad_output, "grad_output", 4), k = checked(kernel, "kernel", 4);
    same_device(go, k);
    const int64_t N = go.size(0), OC = go.size(1), OH = go.size(2), OW = go.size(3);
    const int64_t IC = k.size(1), KH = k.size(2), KW = k.size(3);
    TORCH_CHECK(k.size(0) == OC, "conv2d_grad_input: grad_output has ", OC, " channels, kernel has ", k.size(0));
    const DeviceGuard guard(go.device());
    auto out = torch::empty({N, IC, H, W}, go.options());
    const Scratch work(repdl_hip_conv2d_grad_input_workspace_bytes(go.data_ptr<float>(), k.data_ptr<float>(), N, OC, OH, OW, IC, KH,
                                                                   KW, H, W, sH, sW, pH, pW),
                       go);
    ok(repdl_hip_conv2d_grad_input_ws(go.data_ptr<float>(), k.data_ptr<float>(), out.data_ptr<float>(), N, OC, OH, OW, IC,
                                      KH, KW, H, W, sH, sW, pH, pW, work.ptr(), work.bytes, current_stream()),
       "repdl_hip_conv2d_grad_input_ws");
    return out;
}

torch::Tensor conv2d_grad_kernel(const torch::Tensor &grad_output, const torch::Tensor &input, int64_t KH, int64_t KW,
                                 int64_t sH, int64_t sW, int64_t pH, int64_t pW)
{
    const auto go = checked(grad_output, "grad_output", 4), x = checked(input, "input", 4);
    same_device(go, x);
    const int64_t N = x.size(0), IC = x.size(1), H = x.size(2), W = x.size(3);
    const int64_t OC = go.size(1), OH = go.size(2), OW = go.size(3);
    TORCH_CHECK(go.size(0) == N, "conv2d_grad_kernel: batch sizes differ (", N, " vs ", go.size(0), ")");
    const DeviceGuard guard(x.device());
    auto out = torch::empty({OC, IC, KH, KW}, x.options());
    const Scratch work(repdl_hip_conv2d_grad_kernel_workspace_bytes(go.data_ptr<float>(), x.data_ptr<float>(), N, IC, H, W, OC, OH,
                                                                    OW, KH, KW, sH, sW, pH, pW),
                       x);
    ok(repdl_hip_conv2d_grad_kernel_ws(go.data_ptr<float>(), x.data_ptr<float>(), out.data_ptr<float>(), N, IC, H, W, OC,
                                       OH, OW, KH, KW, sH, sW, pH, pW, work.ptr(), work.bytes, current_stream()),
       "repdl_hip_conv2d_grad_kernel_ws");
    return out;
}

torch::Tensor sum1d(const torch::Tensor &input, bool average)
{
    const auto x = checked(input, "input", 1);
    const int64_t n = x.size(0);
    const DeviceGuard guard(x.device());
    auto out = torch::empty({}, x.options());
    // scratch for the parallel evaluation of the sequential chain
    const Scratch work(repdl_hip_sum1d_workspace_bytes(n), x);
    ok(repdl_hip_sum1d_ws(x.data_ptr<float>(), out.data_ptr<float>(), n, average, work.ptr(), work.bytes, current_stream()),
       "repdl_hip_sum1d_ws");
    return out;
}

torch::Tensor sum2d_dim0(const torch::Tensor &input, bool keepdim, bool average)
{
    const auto x = checked(input, "input", 2);
    const DeviceGuard guard(x.device());
    auto out = torch::empty({1, x.size(1)}, x.options());
    ok(repdl_hip_sum2d_dim0(x.data_ptr<float>(), out.data_ptr<float>(), x.size(0), x.size(1), average, current_stream()),
       "repdl_hip_sum2d_dim0");
    return keepdim ? out : out.squeeze();
}

torch::Tensor sum2d_dim1(const torch::Tensor &input, bool keepdim, bool average)
{
    const auto x = checked(input, "input", 2);
    const DeviceGuard guard(x.device());
    auto out = torch::empty({x.size(0), 1}, x.options());
    const Scratch work(repdl_hip_sum2d_dim1_workspace_bytes(x.size(0), x.size(1)), x);
    ok(repdl_hip_sum2d_dim1_ws(x.data_ptr<float>(), out.data_ptr<float>(), x.size(0), x.size(1), average, work.ptr(), work.bytes,
                               current_stream()),
       "repdl_hip_sum2d_dim1_ws");
    return keepdim ? out : out.squeeze();
}

torch::Tensor sum4d_dim023(const torch::Tensor &input, bool keepdim, bool average)
{
    const auto x = checked(input, "input", 4);
    const DeviceGuard guard(x.device());
    auto out = torch::empty({1, x.size(1), 1, 1}, x.options());
    const Scratch work(repdl_hip_sum4d_dim023_workspace_bytes(x.size(0), x.size(1), x.size(2), x.size(3)), x);
    ok(repdl_hip_sum4d_dim023_ws(x.data_ptr<float>(), out.data_ptr<float>(), x.size(0), x.size(1), x.size(2), x.size(3),
                                 average, work.ptr(), work.bytes, current_stream()),
       "repdl_hip_sum4d_dim023_ws");
    return keepdim ? out : out.squeeze();
}

namespace
{
template <typename F>
torch::Tensor unary(const torch::Tensor &input, F fn, const char *what)
{
    const auto x = checked(input, "input", -1);
    const DeviceGuard guard(x.device());
    auto out = torch::empty_like(x);
    ok(fn(x.data_ptr<float>(), out.data_ptr<float>(), x.numel(), current_stream()), what);
    return out;
}
} // namespace

torch::Tensor exp(const torch::Tensor &input) { return unary(input, repdl_hip_exp, "repdl_hip_exp"); }
torch::Tensor log(const torch::Tensor &input) { return unary(input, repdl_hip_log, "repdl_hip_log"); }
torch::Tensor sqrt(const torch::Tensor &input) { return unary(input, repdl_hip_sqrt, "repdl_hip_sqrt"); }

torch::Tensor div_scalar(const torch::Tensor &input, double other)
{
    const auto x = checked(input, "input", -1);
    const DeviceGuard guard(x.device());
    auto out = torch::empty_like(x);
    ok(repdl_hip_div_scalar(x.data_ptr<float>(), (float)other, out.data_ptr<float>(), x.numel(), current_stream()),
       "repdl_hip_div_scalar");
    return out;
}

// input / other elementwise; `other` is broadcast to the common shape; a 0-dim `other` goes
// through the scalar entry point (repdl/ops.py:98-103 divides by Python numbers and tensors alike)
torch::Tensor div(const torch::Tensor &input, const torch::Tensor &other)
{
    if (other.dim() == 0)
        return div_scalar(input, other.item<double>());
    auto x = checked(input, "input", -1), y = checked(other, "other", -1);
    same_device(x, y);
    const auto shape = at::infer_size(x.sizes(), y.sizes());
    x = x.expand(shape).contiguous();
    y = y.expand(shape).contiguous();
    const DeviceGuard guard(x.device());
    auto out = torch::empty(shape, x.options());
    ok(repdl_hip_div(x.data_ptr<float>(), y.data_ptr<float>(), out.data_ptr<float>(), out.numel(), current_stream()),
       "repdl_hip_div");
    return out;
}

torch::Tensor softmax(const torch::Tensor &input)
{
    const auto x = checked(input, "input", 2);
    const DeviceGuard guard(x.device());
    auto out = torch::empty_like(x);
    ok(repdl_hip_softmax(x.data_ptr<float>(), out.data_ptr<float>(), x.size(0), x.size(1), current_stream()),
       "repdl_hip_softmax");
    return out;
}

torch::Tensor cross_entropy(const torch::Tensor &input, const torch::Tensor &target)
{
    const auto x = checked(input, "input", 2), t = checked(target, "target", 1, torch::kLong);
    same_device(x, t);
    TORCH_CHECK(t.size(0) == x.size(0), "cross_entropy: ", x.size(0), " rows but ", t.size(0), " targets");
    const DeviceGuard guard(x.device());
    auto out = torch::empty({}, x.options());
    // the row losses and the scratch of their mean
    const Scratch work(repdl_hip_cross_entropy_workspace_bytes(x.size(0), x.size(1)), x);
    ok(repdl_hip_cross_entropy_ws(x.data_ptr<float>(), t.data_ptr<int64_t>(), out.data_ptr<float>(), x.size(0), x.size(1),
                                  work.ptr(), work.bytes, current_stream()),
       "repdl_hip_cross_entropy_ws");
    return out;
}
namespace
{
// [N,C,H,W] or [B,F] with per-channel vectors -> outer, channels, inner
void bn_geometry(const torch::Tensor &x, std::initializer_list<torch::Tensor> vectors, int64_t &outer, int64_t &channels,
                 int64_t &inner)
{
    TORCH_CHECK(x.dim() == 4 || x.dim() == 2, "batch norm takes 2-D or 4-D tensors, got ", x.dim(), " dimensions");
    outer = x.size(0);
    channels = x.size(1);
    inner = x.dim() == 4 ? x.size(2) * x.size(3) : 1;
    for (const auto &v : vectors)
    {
        TORCH_CHECK(v.numel() == channels, "a per-channel vector has ", v.numel(), " elements for ", channels, " channels");
        same_device(v, x);
    }
}
} // namespace

// ((input - mean) / std) * weight + bias per channel, every operation rounded (repdl/nn/batchnorm.py:25-32)
torch::Tensor bn_apply(const torch::Tensor &input, const torch::Tensor &mean, const torch::Tensor &std,
                       const torch::Tensor &weight, const torch::Tensor &bias)
{
    const auto x = checked(input, "input", -1);
    const auto m = checked(mean, "mean", 1), s = checked(std, "std", 1), w = checked(weight, "weight", 1),
               b = checked(bias, "bias", 1);
    int64_t outer, channels, inner;
    bn_geometry(x, {m, s, w, b}, outer, channels, inner);
    const DeviceGuard guard(x.device());
    auto out = torch::empty_like(x);
    ok(repdl_hip_bn_apply(x.data_ptr<float>(), m.data_ptr<float>(), s.data_ptr<float>(), w.data_ptr<float>(),
                          b.data_ptr<float>(), out.data_ptr<float>(), outer, channels, inner, current_stream()),
       "repdl_hip_bn_apply");
    return out;
}

// (grad_output * (mean - input)) * coef per channel: what grad_var sums (repdl/nn/batchnorm.py:56-58)
torch::Tensor bn_gvar_term(const torch::Tensor &grad_output, const torch::Tensor &input, const torch::Tensor &mean,
                           const torch::Tensor &coef)
{
    const auto g = checked(grad_output, "grad_output", -1), x = checked(input, "input", -1);
    const auto m = checked(mean, "mean", 1), c = checked(coef, "coef", 1);
    TORCH_CHECK(g.sizes() == x.sizes(), "grad_output and input differ in shape");
    same_device(g, x);
    int64_t outer, channels, inner;
    bn_geometry(x, {m, c}, outer, channels, inner);
    const DeviceGuard guard(x.device());
    auto out = torch::empty_like(x);
    ok(repdl_hip_bn_gvar_term(g.data_ptr<float>(), x.data_ptr<float>(), m.data_ptr<float>(), c.data_ptr<float>(),
                              out.data_ptr<float>(), outer, channels, inner, current_stream()),
       "repdl_hip_bn_gvar_term");
    return out;
}

// ((input - mean) / std) * grad_output per channel: what grad_weight sums (repdl/nn/batchnorm.py:60-61)
torch::Tensor bn_gweight_term(const torch::Tensor &input, const torch::Tensor &mean, const torch::Tensor &std,
                              const torch::Tensor &grad_output)
{
    const auto x = checked(input, "input", -1), g = checked(grad_output, "grad_output", -1);
    const auto m = checked(mean, "mean", 1), s = checked(std, "std", 1);
    TORCH_CHECK(g.sizes() == x.sizes(), "grad_output and input differ in shape");
    same_device(g, x);
    int64_t outer, channels, inner;
    bn_geometry(x, {m, s}, outer, channels, inner);
    const DeviceGuard guard(x.device());
    auto out = torch::empty_like(x);
    ok(repdl_hip_bn_gweight_term(x.data_ptr<float>(), m.data_ptr<float>(), s.data_ptr<float>(), g.data_ptr<float>(),
                                 out.data_ptr<float>(), outer, channels, inner, current_stream()),
       "repdl_hip_bn_gweight_term");
    return out;
}

namespace
{
// the element types of the operators below, by their code in the C ABI
int dtype_code(const torch::Tensor &t, const char *name)
{
    const auto k = t.scalar_type();
    TORCH_CHECK(k == torch::kFloat || k == torch::kBFloat16 || k == torch::kHalf, name, " must be float32, bfloat16 or float16, got ", k);
    return k == torch::kFloat ? REPDL_F32 : k == torch::kBFloat16 ? REPDL_BF16 : REPDL_F16;
}

torch::Tensor checked_any(const torch::Tensor &t, const char *name)
{
    TORCH_CHECK(t.is_cuda(), name, " must be on the GPU (this backend has no CPU path)");
    dtype_code(t, name);
    return t.contiguous();
}

// weight or bias of a layer norm: [n] of the input's type or float32 on the same device, or none
const void *norm_param(const c10::optional<torch::Tensor> &p, torch::Tensor &hold, const char *name, const torch::Tensor &x, int64_t n,
                       int &code)
{
    if (!p.has_value())
        return nullptr;
    hold = checked_any(*p, name);
    same_device(hold, x);
    TORCH_CHECK(hold.numel() == n, name, " has ", hold.numel(), " elements for rows of ", n);
    const int c = dtype_code(hold, name);
    TORCH_CHECK(c == REPDL_F32 || hold.scalar_type() == x.scalar_type(), name, " must be ", x.scalar_type(), " like the input, or float32");
    TORCH_CHECK(code < 0 || code == c, "weight and bias differ in type");
    code = c;
    return hold.data_ptr();
}

int64_t norm_rows(const torch::Tensor &x, int64_t n)
{
    TORCH_CHECK(n >= 0 && (n == 0 ? x.numel() == 0 : x.numel() % n == 0), "layer_norm: ", x.numel(), " elements are no whole rows of ", n);
    return n == 0 ? 0 : x.numel() / n;
}
} // namespace

// rows of n elements normalised; with `stats` also mean and rstd of every row (else undefined)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> layer_norm(const torch::Tensor &input, int64_t n,
                                                                   const c10::optional<torch::Tensor> &weight,
                                                                   const c10::optional<torch::Tensor> &bias, double eps, bool stats)
{
    const auto x = checked_any(input, "input");
    const int64_t rows = norm_rows(x, n);
    const DeviceGuard guard(x.device());
    torch::Tensor hw, hb, mean, rstd;
    int code = -1;
    const void *w = norm_param(weight, hw, "weight", x, n, code), *b = norm_param(bias, hb, "bias", x, n, code);
    auto out = torch::empty_like(x);
    if (stats)
    {
        mean = torch::empty({rows}, x.options().dtype(torch::kFloat));
        rstd = torch::empty({rows}, x.options().dtype(torch::kFloat));
    }
    ok(repdl_hip_layer_norm(x.data_ptr(), w, b, out.data_ptr(), stats ? mean.data_ptr<float>() : nullptr,
                            stats ? rstd.data_ptr<float>() : nullptr, rows, n, (float)eps, dtype_code(x, "input"),
                            code < 0 ? REPDL_F32 : code, current_stream()),
       "repdl_hip_layer_norm");
    return {out, mean, rstd};
}

// the gradients of layer_norm that are asked for (the others are undefined); those of weight and bias are [n], of param_like's type
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> layer_norm_grad(const torch::Tensor &grad_output, const torch::Tensor &input,
                                                                        const torch::Tensor &mean, const torch::Tensor &rstd, int64_t n,
                                                                        const c10::optional<torch::Tensor> &weight,
                                                                        const c10::optional<torch::Tensor> &param_like, bool need_input,
                                                                        bool need_weight, bool need_bias)
{
    const auto x = checked_any(input, "input"), gy = checked_any(grad_output, "grad_output");
    TORCH_CHECK(gy.sizes() == x.sizes() && gy.scalar_type() == x.scalar_type(), "grad_output and input differ in shape or type");
    same_device(gy, x);
    const int64_t rows = norm_rows(x, n);
    const auto m = checked(mean, "mean", 1), r = checked(rstd, "rstd", 1);
    TORCH_CHECK(m.size(0) == rows && r.size(0) == rows, "mean and rstd are not those of the input's ", rows, " rows");
    same_device(m, x);
    same_device(r, x);
    const DeviceGuard guard(x.device());
    torch::Tensor hw, hp, gx, gw, gb;
    int code = -1;
    const void *w = norm_param(weight, hw, "weight", x, n, code);
    norm_param(param_like, hp, "param_like", x, n, code);
    const auto kind = code < 0 ? torch::kFloat : code == REPDL_F32 ? torch::kFloat : x.scalar_type();
    if (need_input)
        gx = torch::empty_like(x);
    if (need_weight)
        gw = torch::empty({n}, x.options().dtype(kind));
    if (need_bias)
        gb = torch::empty({n}, x.options().dtype(kind));
    const Scratch work(need_weight || need_bias ? repdl_hip_layer_norm_grad_workspace_bytes(rows, n) : 0, x);
    ok(repdl_hip_layer_norm_grad_ws(gy.data_ptr(), x.data_ptr(), w, m.data_ptr<float>(), r.data_ptr<float>(),
                                    need_input ? gx.data_ptr() : nullptr, need_weight ? gw.data_ptr() : nullptr,
                                    need_bias ? gb.data_ptr() : nullptr, rows, n, dtype_code(x, "input"), code < 0 ? REPDL_F32 : code,
                                    work.ptr(), work.bytes, current_stream()),
       "repdl_hip_layer_norm_grad_ws");
    return {gx, gw, gb};
}

namespace
{
const int64_t *dropout_state(const torch::Tensor &state)
{
    TORCH_CHECK(state.is_cuda() && state.scalar_type() == torch::kLong && state.dim() == 1 && state.size(0) == 2 && state.is_contiguous(),
                "the state of dropout is an int64 tensor (seed, call) on the GPU");
    return state.data_ptr<int64_t>();
}
} // namespace

// dropout (added to residual, if there is one) for the call (seed, call), read from `state` on the device where there is one
torch::Tensor dropout(const torch::Tensor &input, const c10::optional<torch::Tensor> &residual, double p,
                      const c10::optional<torch::Tensor> &state, uint64_t seed, uint64_t call)
{
    const auto x = checked_any(input, "input");
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "dropout probability has to be between 0 and 1, but got ", p);
    torch::Tensor r;
    if (residual.has_value())
    {
        r = checked_any(*residual, "residual");
        same_device(r, x);
        TORCH_CHECK(r.sizes() == x.sizes() && r.scalar_type() == x.scalar_type(), "residual and input differ in shape or type");
    }
    if (state.has_value())
        same_device(*state, x);
    const DeviceGuard guard(x.device());
    auto out = torch::empty_like(x);
    ok(repdl_hip_dropout(x.data_ptr(), r.defined() ? r.data_ptr() : nullptr, out.data_ptr(), x.numel(), p,
                         state.has_value() ? dropout_state(*state) : nullptr, seed, call, dtype_code(x, "input"), current_stream()),
       "repdl_hip_dropout");
    return out;
}

// a copy of `state`, whose call number is then one more
torch::Tensor dropout_next_call(const torch::Tensor &state)
{
    dropout_state(state);
    const DeviceGuard guard(state.device());
    auto used = torch::empty_like(state);
    ok(repdl_hip_dropout_next_call(state.data_ptr<int64_t>(), used.data_ptr<int64_t>(), current_stream()), "repdl_hip_dropout_next_call");
    return used;
}

namespace
{
// logits of a preference loss: rows of contiguous elements, any strides between sequences and steps
torch::Tensor pref_logits(const torch::Tensor &logits, const torch::Tensor &target)
{
    TORCH_CHECK(logits.is_cuda(), "logits must be on the GPU (this backend has no CPU path)");
    dtype_code(logits, "logits");
    TORCH_CHECK(logits.dim() == 3, "logits must have 3 dimensions (sequence, step, vocabulary), got ", logits.dim());
    TORCH_CHECK(logits.size(0) >= 2 && logits.size(0) % 2 == 0, "logits: the preferred answers, then as many others (got ", logits.size(0),
                " sequences)");
    TORCH_CHECK(logits.size(2) >= 1, "logits: an empty vocabulary");
    TORCH_CHECK(target.is_cuda() && target.scalar_type() == torch::kLong, "target must be int64 on the GPU");
    TORCH_CHECK(target.dim() == 2 && target.size(0) == logits.size(0) && target.size(1) == logits.size(1), "target must be [", logits.size(0),
                ", ", logits.size(1), "] like the logits' rows");
    same_device(target, logits);
    return logits.stride(2) == 1 || logits.size(2) == 1 ? logits : logits.contiguous();
}
} // namespace

// loss, log probabilities of the sequences, and (with `grad`) row statistics and coefficients for the backward pass
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> preference_loss(const torch::Tensor &logits, const torch::Tensor &target,
                                                                                       const c10::optional<torch::Tensor> &ref_logps,
                                                                                       double beta, double label_smoothing,
                                                                                       int64_t ignore_index, bool grad)
{
    const auto x = pref_logits(logits, target), t = target.contiguous();
    const int64_t seqs = x.size(0), steps = x.size(1), vocab = x.size(2);
    torch::Tensor ref, stats, coef;
    if (ref_logps.has_value())
    {
        ref = checked(*ref_logps, "ref_logps", 1);
        same_device(ref, x);
        TORCH_CHECK(ref.size(0) == seqs, "ref_logps has ", ref.size(0), " elements for ", seqs, " sequences");
    }
    const DeviceGuard guard(x.device());
    const auto f32 = x.options().dtype(torch::kFloat);
    auto loss = torch::empty({}, f32), logps = torch::empty({seqs}, f32);
    if (grad)
    {
        stats = torch::empty({seqs, steps, 2}, f32);
        coef = torch::empty({seqs}, f32);
    }
    const Scratch work(repdl_hip_preference_loss_workspace_bytes(seqs / 2, steps, vocab), x);
    ok(repdl_hip_preference_loss_ws(x.data_ptr(), t.data_ptr<int64_t>(), ref.defined() ? ref.data_ptr<float>() : nullptr,
                                    loss.data_ptr<float>(), logps.data_ptr<float>(), grad ? stats.data_ptr<float>() : nullptr,
                                    grad ? coef.data_ptr<float>() : nullptr, seqs / 2, steps, vocab, x.stride(0), x.stride(1), beta,
                                    label_smoothing, ignore_index, dtype_code(x, "logits"), work.ptr(), work.bytes, current_stream()),
       "repdl_hip_preference_loss_ws");
    return {loss, logps, stats, coef};
}

torch::Tensor preference_loss_grad(const torch::Tensor &logits, const torch::Tensor &target, const torch::Tensor &row_stats,
                                   const torch::Tensor &coef, const torch::Tensor &grad_loss, int64_t ignore_index)
{
    const auto x = pref_logits(logits, target), t = target.contiguous();
    const int64_t seqs = x.size(0), steps = x.size(1), vocab = x.size(2);
    const auto st = checked(row_stats, "row_stats", 3), c = checked(coef, "coef", 1), g = checked(grad_loss, "grad_loss", 0);
    TORCH_CHECK(st.size(0) == seqs && st.size(1) == steps && st.size(2) == 2 && c.size(0) == seqs,
                "row_stats and coef are not those of these logits");
    same_device(st, x);
    same_device(c, x);
    same_device(g, x);
    const DeviceGuard guard(x.device());
    auto out = torch::empty({seqs, steps, vocab}, x.options());
    ok(repdl_hip_preference_loss_grad(x.data_ptr(), t.data_ptr<int64_t>(), st.data_ptr<float>(), c.data_ptr<float>(), g.data_ptr<float>(),
                                      out.data_ptr(), seqs / 2, steps, vocab, x.stride(0), x.stride(1), ignore_index,
                                      dtype_code(x, "logits"), current_stream()),
       "repdl_hip_preference_loss_grad");
    return out;
}

// ---- autograd ---------------------------------------------------------------------------------
// The differentiable forms that repdl_amd/nn/functional.py serves: the same calls and the same gradients as its Python
// functions, recorded and run without the interpreter.  (Forward and backward of dropout on 64000 elements: 52 us of host time
// against 63 through Python functions over this binding; 37 are torch.autograd.grad's own.)
namespace
{
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients of a function that is differentiable once: where the backward pass is recorded, differentiating them again is an
// error, not a silent zero.
variable_list once(variable_list grads)
{
    if (!at::GradMode::is_enabled())
        return grads;
    for (auto &g : grads)
        if (g.defined())
            g = g.detach().requires_grad_(true);
    auto error = std::make_shared<torch::autograd::DelayedError>("this function can be differentiated only once", grads.size());
    return (*error)(std::move(grads));
}

// A leaf's gradient accumulator belongs to the stream of the first graph that used the leaf, for as long as a graph of it lives.
// If that is the default stream, a backward pass through the leaf under capture makes the default stream wait for an event of the
// capture, which ends the process inside PyTorch's engine.  Said here, in the forward pass, where it can still be an error.
void refuse_eager_leaf(const torch::Tensor &t, const char *name)
{
    if (!at::GradMode::is_enabled() || !t.defined() || !t.is_cuda() || !t.requires_grad() || !t.is_leaf())
        return;
    const auto current = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index());
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (current.stream() == nullptr || hipStreamIsCapturing(current.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone)
        return;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto held = node ? node->stream() : c10::nullopt;
    TORCH_CHECK(!held.has_value() || *held != c10::Stream(c10::Stream::DEFAULT, t.device()), name,
                " still belongs to an eager graph of the default stream: a backward pass cannot be captured beside it; delete the eager "
                "graph's results first (or run the eager steps on a side stream)");
}

struct LayerNormFunction : public torch::autograd::Function<LayerNormFunction>
{
    static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &x, const c10::optional<torch::Tensor> &weight,
                                 const c10::optional<torch::Tensor> &bias, int64_t n, double eps)
    {
        auto r = layer_norm(x, n, weight, bias, eps, true);
        // (a bias alone: for its type)
        ctx->save_for_backward({x, weight.has_value() ? *weight : torch::Tensor(), !weight.has_value() && bias.has_value() ? *bias : torch::Tensor(),
                                std::get<1>(r), std::get<2>(r)});
        ctx->saved_data["n"] = n;
        ctx->saved_data["weight"] = weight.has_value();
        ctx->saved_data["bias"] = bias.has_value();
        if (weight.has_value())
            ctx->saved_data["shape"] = weight->sizes().vec();
        else if (bias.has_value())
            ctx->saved_data["shape"] = bias->sizes().vec();
        return std::get<0>(r);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        const auto saved = ctx->get_saved_variables();
        const bool has_w = ctx->saved_data["weight"].toBool(), has_b = ctx->saved_data["bias"].toBool();
        // (the edges of the graph are those of the tensors that were there)
        const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1),
                   need_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
        const auto opt = [](const torch::Tensor &t) { return t.defined() ? c10::optional<torch::Tensor>(t) : c10::nullopt; };
        auto r = layer_norm_grad(grads[0], saved[0], saved[3], saved[4], ctx->saved_data["n"].toInt(), opt(saved[1]), opt(saved[2]), need_x,
                                 need_w, need_b);
        auto gw = std::get<1>(r), gb = std::get<2>(r);
        if (gw.defined())
            gw = gw.view(ctx->saved_data["shape"].toIntVector());
        if (gb.defined())
            gb = gb.view(ctx->saved_data["shape"].toIntVector());
        return once({std::get<0>(r), gw, gb, torch::Tensor(), torch::Tensor()});
    }
};

struct DropoutFunction : public torch::autograd::Function<DropoutFunction>
{
    static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &x, const c10::optional<torch::Tensor> &residual, double p,
                                 const c10::optional<torch::Tensor> &state, int64_t seed, int64_t call)
    {
        if (state.has_value())
            ctx->save_for_backward({*state});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["call"] = call;
        ctx->saved_data["state"] = state.has_value();
        ctx->saved_data["residual"] = residual.has_value();
        return dropout(x, residual, p, state, (uint64_t)seed, (uint64_t)call);
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        c10::optional<torch::Tensor> state;
        if (ctx->saved_data["state"].toBool())
            state = ctx->get_saved_variables()[0];
        torch::Tensor gx, gr;
        if (ctx->needs_input_grad(0)) // the mask again, from the same call of the generator
            gx = dropout(grads[0], c10::nullopt, ctx->saved_data["p"].toDouble(), state, (uint64_t)ctx->saved_data["seed"].toInt(),
                         (uint64_t)ctx->saved_data["call"].toInt());
        if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1))
            gr = grads[0];
        return once({gx, gr, torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()});
    }
};

struct PreferenceFunction : public torch::autograd::Function<PreferenceFunction>
{
    static variable_list forward(AutogradContext *ctx, const torch::Tensor &logits, const torch::Tensor &target,
                                 const c10::optional<torch::Tensor> &ref_logps, double beta, double label_smoothing, int64_t ignore_index)
    {
        auto r = preference_loss(logits, target, ref_logps, beta, label_smoothing, ignore_index, true);
        ctx->save_for_backward({logits, target, std::get<2>(r), std::get<3>(r)});
        ctx->saved_data["ignore"] = ignore_index;
        ctx->mark_non_differentiable({std::get<1>(r)});
        ctx->set_materialize_grads(false);
        return {std::get<0>(r), std::get<1>(r)};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        torch::Tensor g;
        if (grads[0].defined())
        {
            const auto saved = ctx->get_saved_variables();
            g = preference_loss_grad(saved[0], saved[1], saved[2], saved[3], grads[0], ctx->saved_data["ignore"].toInt());
        }
        return once({g, torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()});
    }
};
} // namespace

torch::Tensor layer_norm_autograd(const torch::Tensor &input, int64_t n, const c10::optional<torch::Tensor> &weight,
                                  const c10::optional<torch::Tensor> &bias, double eps)
{
    refuse_eager_leaf(input, "input");
    if (weight.has_value())
        refuse_eager_leaf(*weight, "weight");
    if (bias.has_value())
        refuse_eager_leaf(*bias, "bias");
    return LayerNormFunction::apply(input, weight, bias, n, eps);
}

torch::Tensor dropout_autograd(const torch::Tensor &input, const c10::optional<torch::Tensor> &residual, double p,
                               const c10::optional<torch::Tensor> &state, uint64_t seed, uint64_t call)
{
    refuse_eager_leaf(input, "input");
    if (residual.has_value())
        refuse_eager_leaf(*residual, "residual");
    return DropoutFunction::apply(input, residual, p, state, (int64_t)seed, (int64_t)call);
}

std::tuple<torch::Tensor, torch::Tensor> preference_loss_autograd(const torch::Tensor &logits, const torch::Tensor &target,
                                                                  const c10::optional<torch::Tensor> &ref_logps, double beta,
                                                                  double label_smoothing, int64_t ignore_index)
{
    refuse_eager_leaf(logits, "logits");
    auto r = PreferenceFunction::apply(logits, target, ref_logps, beta, label_smoothing, ignore_index);
    return {r[0], r[1]};
}

} // namespace hip
} // namespace repdl

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    namespace h = repdl::hip;
    // Importing the module touches no device.  The one-time check of the matrix instructions runs inside the
    // first GEMM-shaped call on a device, or when the program calls init() -- which a program that captures
    // graphs does before its first capture (a check cannot run under capture).
    m.def("init", []() {
        const int rc = repdl_hip_init();
        TORCH_CHECK(rc == 0, "repdl_hip_init failed with code ", rc, ": ", repdl_hip_error_string(rc));
    });
    m.def("conv2d", &h::conv2d);
    m.def("conv2d_grad_input", &h::conv2d_grad_input);
    m.def("conv2d_grad_kernel", &h::conv2d_grad_kernel);
    m.def("cross_entropy", &h::cross_entropy);
    m.def("mm", &h::mm);
    m.def("softmax", &h::softmax);
    m.def("sum1d", &h::sum1d, py::arg("input"), py::arg("average") = false);
    m.def("sum2d_dim0", &h::sum2d_dim0, py::arg("input"), py::arg("keepdim") = false, py::arg("average") = false);
    m.def("sum2d_dim1", &h::sum2d_dim1, py::arg("input"), py::arg("keepdim") = false, py::arg("average") = false);
    m.def("sum4d_dim023", &h::sum4d_dim023, py::arg("input"), py::arg("keepdim") = false, py::arg("average") = false);
    m.def("exp", &h::exp);
    m.def("log", &h::log);
    m.def("sqrt", &h::sqrt);
    m.def("div", &h::div);
    m.def("div_scalar", &h::div_scalar);
    m.def("mm_bias", &h::mm_bias);
    m.def("conv2d_bias", &h::conv2d_bias);
    m.def("bn_apply", &h::bn_apply);
    m.def("bn_gvar_term", &h::bn_gvar_term);
    m.def("bn_gweight_term", &h::bn_gweight_term);
    m.def("layer_norm", &h::layer_norm);
    m.def("layer_norm_grad", &h::layer_norm_grad);
    m.def("dropout", &h::dropout);
    m.def("dropout_next_call", &h::dropout_next_call);
    m.def("preference_loss", &h::preference_loss);
    m.def("preference_loss_grad", &h::preference_loss_grad);
    m.def("layer_norm_autograd", &h::layer_norm_autograd);
    m.def("dropout_autograd", &h::dropout_autograd);
    m.def("preference_loss_autograd", &h::preference_loss_autograd);
}
