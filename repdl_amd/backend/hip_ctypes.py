"""``repdl_amd.backend.hip_ctypes`` -- the function set of RepDL's compiled
``repdl.backend.cuda`` (backend/cuda/bind.cpp:12-19) bound to the C ABI with ctypes:
the same ten functions with the same positional signatures, tensors in and a new
tensor out, plus the elementwise operators (``exp``, ``log``, ``sqrt``, ``div``,
``div_scalar``), ``mm_bias`` / ``conv2d_bias`` (the layer's bias added in the
kernel's epilogue), the fused elementwise passes of batch normalisation, and layer
normalisation, dropout and the preference loss.  ``repdl_amd.backend.hip`` serves these when the compiled binding
(csrc/bind.cpp) has not been built; both call the same library.

Each function validates its tensors (float32, on the GPU, made contiguous),
allocates the output with PyTorch on the input's device and hands raw pointers
and the current stream to the C ABI (include/repdl_hip.h).  Output shapes follow
the reference, including ``squeeze()`` of the sums when ``keepdim`` is false
(backend/cuda/summation.cu:41, 68, 103, 141) and the 0-dim results of ``sum1d``
and ``cross_entropy``.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from .. import _lib

_P = ctypes.c_void_p


def _check(t: torch.Tensor, name: str, dim: int | None = None, dtype=torch.float32) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor" % name)
    if not t.is_cuda:
        raise RuntimeError("%s must be on the GPU (this backend has no CPU path)" % name)
    if t.dtype != dtype:
        raise RuntimeError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if dim is not None and t.dim() != dim:
        raise RuntimeError("%s must have %d dimensions, got %d" % (name, dim, t.dim()))
    return t.contiguous()


def _ptr(t: torch.Tensor) -> _P:
    return _P(t.data_ptr())


def _stream(t: torch.Tensor) -> _P:
    return _P(torch.cuda.current_stream(t.device).cuda_stream)


def _scratch(query: str, like: torch.Tensor, *args):
    """Scratch memory of a call from PyTorch's allocator, sized by the entry point's own query: (tensor or None,
    pointer, size).  The library then allocates, frees and keeps nothing, so the call can be captured into a graph."""
    nbytes = int(getattr(_lib.lib(), query)(*args))
    if nbytes == 0:
        return None, None, ctypes.c_size_t(0)
    work = torch.empty((nbytes,), dtype=torch.uint8, device=like.device)
    return work, _ptr(work), ctypes.c_size_t(nbytes)


def _same_device(a: torch.Tensor, b: torch.Tensor) -> None:
    if a.device != b.device:
        raise RuntimeError("tensors are on different devices: %s and %s" % (a.device, b.device))


def _bias(bias, like: torch.Tensor, channels: int):
    """The bias of a layer as a pointer: [channels] on the same device, or None."""
    if bias is None:
        return None, None
    b = _check(bias, "bias", 1)
    _same_device(b, like)
    if b.shape[0] != channels:
        raise RuntimeError("bias has %d elements for %d output channels" % (b.shape[0], channels))
    return b, _ptr(b)


def mm(input: torch.Tensor, mat2: torch.Tensor, transA: bool, transB: bool) -> torch.Tensor:
    return mm_bias(input, mat2, None, transA, transB)


def mm_bias(input: torch.Tensor, mat2: torch.Tensor, bias, transA: bool, transB: bool) -> torch.Tensor:
    """mm followed by ``+= bias`` (repdl/nn/linear.py:21-22), the addition made in the kernel's epilogue."""
    a, b = _check(input, "input", 2), _check(mat2, "mat2", 2)
    _same_device(a, b)
    M, K = (a.shape[0], a.shape[1]) if not transA else (a.shape[1], a.shape[0])
    N, Kb = (b.shape[1], b.shape[0]) if not transB else (b.shape[0], b.shape[1])
    if K != Kb:
        raise RuntimeError("mm: inner dimensions differ (%d vs %d)" % (K, Kb))
    hold, bp = _bias(bias, a, N)
    out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    with torch.cuda.device(a.device):
        _lib.call("repdl_hip_mm_bias", _ptr(a), _ptr(b), bp, _ptr(out), M, N, K, int(bool(transA)), int(bool(transB)),
                  _stream(a))
    return out


def conv2d(input, kernel, strideH, strideW, paddingH, paddingW, groups) -> torch.Tensor:
    return conv2d_bias(input, kernel, None, strideH, strideW, paddingH, paddingW, groups)


def conv2d_bias(input, kernel, bias, strideH, strideW, paddingH, paddingW, groups) -> torch.Tensor:
    """conv2d followed by ``+= bias`` per output channel (repdl/nn/conv.py:27-28), in the epilogue."""
    x, k = _check(input, "input", 4), _check(kernel, "kernel", 4)
    _same_device(x, k)
    N, IC, H, W = x.shape
    OC, ICg, KH, KW = k.shape
    if groups <= 0 or IC % groups or OC % groups or ICg != IC // groups:
        raise RuntimeError("conv2d: channels (%d in, %d out, kernel %d) do not match groups=%d" % (IC, OC, ICg, groups))
    if H + 2 * paddingH < KH or W + 2 * paddingW < KW:
        raise RuntimeError("conv2d: kernel larger than padded input")
    OH, OW = (H + 2 * paddingH - KH) // strideH + 1, (W + 2 * paddingW - KW) // strideW + 1
    hold, bp = _bias(bias, x, OC)
    out = torch.empty((N, OC, OH, OW), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        dims = (N, IC, H, W, OC, KH, KW, strideH, strideW, paddingH, paddingW, groups)
        work, wp, wn = _scratch("repdl_hip_conv2d_workspace_bytes", x, _ptr(x), _ptr(k), *dims)
        _lib.call("repdl_hip_conv2d_ws", _ptr(x), _ptr(k), bp, _ptr(out), *dims, wp, wn, _stream(x))
    return out


def conv2d_grad_input(grad_output, kernel, H, W, strideH, strideW, paddingH, paddingW) -> torch.Tensor:
    go, k = _check(grad_output, "grad_output", 4), _check(kernel, "kernel", 4)
    _same_device(go, k)
    N, OC, OH, OW = go.shape
    OCk, IC, KH, KW = k.shape
    if OCk != OC:
        raise RuntimeError("conv2d_grad_input: grad_output has %d channels, kernel has %d" % (OC, OCk))
    out = torch.empty((N, IC, H, W), dtype=torch.float32, device=go.device)
    with torch.cuda.device(go.device):
        dims = (N, OC, OH, OW, IC, KH, KW, H, W, strideH, strideW, paddingH, paddingW)
        work, wp, wn = _scratch("repdl_hip_conv2d_grad_input_workspace_bytes", go, _ptr(go), _ptr(k), *dims)
        _lib.call("repdl_hip_conv2d_grad_input_ws", _ptr(go), _ptr(k), _ptr(out), *dims, wp, wn, _stream(go))
    return out


def conv2d_grad_kernel(grad_output, input, KH, KW, strideH, strideW, paddingH, paddingW) -> torch.Tensor:
    go, x = _check(grad_output, "grad_output", 4), _check(input, "input", 4)
    _same_device(go, x)
    N, IC, H, W = x.shape
    Ng, OC, OH, OW = go.shape
    if Ng != N:
        raise RuntimeError("conv2d_grad_kernel: batch sizes differ (%d vs %d)" % (N, Ng))
    out = torch.empty((OC, IC, KH, KW), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        dims = (N, IC, H, W, OC, OH, OW, KH, KW, strideH, strideW, paddingH, paddingW)
        work, wp, wn = _scratch("repdl_hip_conv2d_grad_kernel_workspace_bytes", x, _ptr(go), _ptr(x), *dims)
        _lib.call("repdl_hip_conv2d_grad_kernel_ws", _ptr(go), _ptr(x), _ptr(out), *dims, wp, wn, _stream(x))
    return out


def sum1d(input, average: bool = False) -> torch.Tensor:
    x = _check(input, "input", 1)
    out = torch.empty((), dtype=torch.float32, device=x.device)
    n = x.shape[0]
    with torch.cuda.device(x.device):
        # scratch for the parallel evaluation of the sequential chain
        work, wp, wn = _scratch("repdl_hip_sum1d_workspace_bytes", x, n)
        _lib.call("repdl_hip_sum1d_ws", _ptr(x), _ptr(out), n, int(bool(average)), wp, wn, _stream(x))
    return out


def sum2d_dim0(input, keepdim: bool = False, average: bool = False) -> torch.Tensor:
    x = _check(input, "input", 2)
    M, N = x.shape
    out = torch.empty((1, N), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.call("repdl_hip_sum2d_dim0", _ptr(x), _ptr(out), M, N, int(bool(average)), _stream(x))
    return out if keepdim else out.squeeze()


def sum2d_dim1(input, keepdim: bool = False, average: bool = False) -> torch.Tensor:
    x = _check(input, "input", 2)
    M, N = x.shape
    out = torch.empty((M, 1), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        work, wp, wn = _scratch("repdl_hip_sum2d_dim1_workspace_bytes", x, M, N)
        _lib.call("repdl_hip_sum2d_dim1_ws", _ptr(x), _ptr(out), M, N, int(bool(average)), wp, wn, _stream(x))
    return out if keepdim else out.squeeze()


def sum4d_dim023(input, keepdim: bool = False, average: bool = False) -> torch.Tensor:
    x = _check(input, "input", 4)
    N, C, H, W = x.shape
    out = torch.empty((1, C, 1, 1), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        work, wp, wn = _scratch("repdl_hip_sum4d_dim023_workspace_bytes", x, N, C, H, W)
        _lib.call("repdl_hip_sum4d_dim023_ws", _ptr(x), _ptr(out), N, C, H, W, int(bool(average)), wp, wn, _stream(x))
    return out if keepdim else out.squeeze()


def _unary(name: str, input: torch.Tensor) -> torch.Tensor:
    x = _check(input, "input")
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.call(name, _ptr(x), _ptr(out), x.numel(), _stream(x))
    return out


def exp(input: torch.Tensor) -> torch.Tensor:
    return _unary("repdl_hip_exp", input)


def log(input: torch.Tensor) -> torch.Tensor:
    return _unary("repdl_hip_log", input)


def sqrt(input: torch.Tensor) -> torch.Tensor:
    return _unary("repdl_hip_sqrt", input)


def div(input: torch.Tensor, other: torch.Tensor) -> torch.Tensor:
    """input / other elementwise; ``other`` is broadcast to ``input``'s shape.  A
    0-dim ``other`` goes through the scalar entry point."""
    x = _check(input, "input")
    if other.dim() == 0:
        return div_scalar(x, float(other))
    y = _check(other, "other")
    _same_device(x, y)
    shape = torch.broadcast_shapes(x.shape, y.shape)
    if tuple(shape) != tuple(x.shape):
        x = x.expand(shape).contiguous()
    if tuple(y.shape) != tuple(shape):
        y = y.expand(shape).contiguous()
    out = torch.empty(shape, dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.call("repdl_hip_div", _ptr(x), _ptr(y), _ptr(out), out.numel(), _stream(x))
    return out


def div_scalar(input: torch.Tensor, other: float) -> torch.Tensor:
    x = _check(input, "input")
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.call("repdl_hip_div_scalar", _ptr(x), ctypes.c_float(other), _ptr(out), x.numel(), _stream(x))
    return out


def softmax(input: torch.Tensor) -> torch.Tensor:
    x = _check(input, "input", 2)
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.call("repdl_hip_softmax", _ptr(x), _ptr(out), x.shape[0], x.shape[1], _stream(x))
    return out


def cross_entropy(input: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
    x = _check(input, "input", 2)
    t = _check(target, "target", 1, dtype=torch.int64)
    _same_device(x, t)
    if t.shape[0] != x.shape[0]:
        raise RuntimeError("cross_entropy: %d rows but %d targets" % (x.shape[0], t.shape[0]))
    out = torch.empty((), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        # the row losses and the scratch of their mean
        work, wp, wn = _scratch("repdl_hip_cross_entropy_workspace_bytes", x, x.shape[0], x.shape[1])
        _lib.call("repdl_hip_cross_entropy_ws", _ptr(x), _ptr(t), _ptr(out), x.shape[0], x.shape[1], wp, wn, _stream(x))
    return out


def _bn_geometry(x: torch.Tensor, *vectors: torch.Tensor):
    """[N,C,H,W] or [B,F] with per-channel vectors of C (F) elements -> (outer, channels, inner)."""
    if x.dim() == 4:
        outer, channels, inner = x.shape[0], x.shape[1], x.shape[2] * x.shape[3]
    elif x.dim() == 2:
        outer, channels, inner = x.shape[0], x.shape[1], 1
    else:
        raise RuntimeError("batch norm takes 2-D or 4-D tensors, got %d dimensions" % x.dim())
    for v in vectors:
        if v.numel() != channels:
            raise RuntimeError("a per-channel vector has %d elements for %d channels" % (v.numel(), channels))
        _same_device(v, x)
    return outer, channels, inner


def bn_apply(input, mean, std, weight, bias) -> torch.Tensor:
    """((input - mean) / std) * weight + bias per channel, every operation rounded (repdl/nn/batchnorm.py:25-32)."""
    x = _check(input, "input")
    m, s, w, b = (_check(t, n, 1) for t, n in ((mean, "mean"), (std, "std"), (weight, "weight"), (bias, "bias")))
    outer, channels, inner = _bn_geometry(x, m, s, w, b)
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.call("repdl_hip_bn_apply", _ptr(x), _ptr(m), _ptr(s), _ptr(w), _ptr(b), _ptr(out), outer, channels, inner,
                  _stream(x))
    return out


def bn_gvar_term(grad_output, input, mean, coef) -> torch.Tensor:
    """(grad_output * (mean - input)) * coef per channel: what grad_var sums (repdl/nn/batchnorm.py:56-58)."""
    g, x = _check(grad_output, "grad_output"), _check(input, "input")
    m, c = _check(mean, "mean", 1), _check(coef, "coef", 1)
    if g.shape != x.shape:
        raise RuntimeError("grad_output and input differ in shape")
    _same_device(g, x)
    outer, channels, inner = _bn_geometry(x, m, c)
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.call("repdl_hip_bn_gvar_term", _ptr(g), _ptr(x), _ptr(m), _ptr(c), _ptr(out), outer, channels, inner, _stream(x))
    return out


def bn_gweight_term(input, mean, std, grad_output) -> torch.Tensor:
    """((input - mean) / std) * grad_output per channel: what grad_weight sums (repdl/nn/batchnorm.py:60-61)."""
    x, g = _check(input, "input"), _check(grad_output, "grad_output")
    m, s = _check(mean, "mean", 1), _check(std, "std", 1)
    if g.shape != x.shape:
        raise RuntimeError("grad_output and input differ in shape")
    _same_device(g, x)
    outer, channels, inner = _bn_geometry(x, m, s)
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.call("repdl_hip_bn_gweight_term", _ptr(x), _ptr(m), _ptr(s), _ptr(g), _ptr(out), outer, channels, inner,
                  _stream(x))
    return out


_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check_any(t: torch.Tensor, name: str) -> torch.Tensor:
    """A tensor of one of the types that layer norm, dropout and the preference loss take."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor" % name)
    if not t.is_cuda:
        raise RuntimeError("%s must be on the GPU (this backend has no CPU path)" % name)
    if t.dtype not in _DTYPES:
        raise RuntimeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    return t.contiguous()


def _opt(t):
    return None if t is None else _ptr(t)


def _norm_param(p, name: str, x: torch.Tensor, n: int, code):
    """weight or bias of a layer norm: [n] of the input's type or float32 on the same device, or None -> tensor, type code"""
    if p is None:
        return None, code
    t = _check_any(p, name)
    _same_device(t, x)
    if t.numel() != n:
        raise RuntimeError("%s has %d elements for rows of %d" % (name, t.numel(), n))
    if t.dtype not in (torch.float32, x.dtype):
        raise RuntimeError("%s must be %s like the input, or float32" % (name, x.dtype))
    if code is not None and code != _DTYPES[t.dtype]:
        raise RuntimeError("weight and bias differ in type")
    return t, _DTYPES[t.dtype]


def _norm_rows(x: torch.Tensor, n: int) -> int:
    if n < 0 or (x.numel() != 0 if n == 0 else x.numel() % n != 0):
        raise RuntimeError("layer_norm: %d elements are no whole rows of %d" % (x.numel(), n))
    return 0 if n == 0 else x.numel() // n


def layer_norm(input, n: int, weight, bias, eps: float, stats: bool):
    """Rows of n elements normalised -> output and, with ``stats``, mean and rstd of every row (else None)."""
    x = _check_any(input, "input")
    rows = _norm_rows(x, n)
    w, code = _norm_param(weight, "weight", x, n, None)
    b, code = _norm_param(bias, "bias", x, n, code)
    out = torch.empty_like(x)
    mean, rstd = (torch.empty((rows,), dtype=torch.float32, device=x.device) if stats else None for _ in range(2))
    with torch.cuda.device(x.device):
        _lib.call("repdl_hip_layer_norm", _ptr(x), _opt(w), _opt(b), _ptr(out), _opt(mean), _opt(rstd), rows, n, eps, _DTYPES[x.dtype],
                  code or 0, _stream(x))
    return out, mean, rstd


def layer_norm_grad(grad_output, input, mean, rstd, n: int, weight, param_like, need_input: bool, need_weight: bool, need_bias: bool):
    """The gradients of layer_norm that are asked for (else None); those of weight and bias are [n], of param_like's type."""
    x, gy = _check_any(input, "input"), _check_any(grad_output, "grad_output")
    if gy.shape != x.shape or gy.dtype != x.dtype:
        raise RuntimeError("grad_output and input differ in shape or type")
    _same_device(gy, x)
    rows = _norm_rows(x, n)
    m, r = _check(mean, "mean", 1), _check(rstd, "rstd", 1)
    if m.shape[0] != rows or r.shape[0] != rows:
        raise RuntimeError("mean and rstd are not those of the input's %d rows" % rows)
    _same_device(m, x)
    _same_device(r, x)
    w, code = _norm_param(weight, "weight", x, n, None)
    _, code = _norm_param(param_like, "param_like", x, n, code)
    kind = x.dtype if code else torch.float32
    gx = torch.empty_like(x) if need_input else None
    gw = torch.empty((n,), dtype=kind, device=x.device) if need_weight else None
    gb = torch.empty((n,), dtype=kind, device=x.device) if need_bias else None
    with torch.cuda.device(x.device):
        work, wp, wn = None, None, ctypes.c_size_t(0)
        if need_weight or need_bias:
            work, wp, wn = _scratch("repdl_hip_layer_norm_grad_workspace_bytes", x, rows, n)
        _lib.call("repdl_hip_layer_norm_grad_ws", _ptr(gy), _ptr(x), _opt(w), _ptr(m), _ptr(r), _opt(gx), _opt(gw), _opt(gb), rows, n,
                  _DTYPES[x.dtype], code or 0, wp, wn, _stream(x))
    return gx, gw, gb


def _dropout_state(state: torch.Tensor) -> _P:
    if not (state.is_cuda and state.dtype == torch.int64 and tuple(state.shape) == (2,) and state.is_contiguous()):
        raise RuntimeError("the state of dropout is an int64 tensor (seed, call) on the GPU")
    return _ptr(state)


def dropout(input, residual, p: float, state, seed: int, call: int) -> torch.Tensor:
    """Dropout (added to residual, if there is one) for the call (seed, call), read from ``state`` on the device where there is one."""
    x = _check_any(input, "input")
    if not 0.0 <= p <= 1.0:
        raise RuntimeError("dropout probability has to be between 0 and 1, but got %s" % p)
    r = None
    if residual is not None:
        r = _check_any(residual, "residual")
        _same_device(r, x)
        if r.shape != x.shape or r.dtype != x.dtype:
            raise RuntimeError("residual and input differ in shape or type")
    if state is not None:
        _same_device(state, x)
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.call("repdl_hip_dropout", _ptr(x), _opt(r), _ptr(out), x.numel(), p, None if state is None else _dropout_state(state), seed, call,
                  _DTYPES[x.dtype], _stream(x))
    return out


def dropout_next_call(state: torch.Tensor) -> torch.Tensor:
    """A copy of ``state``, whose call number is then one more."""
    sp = _dropout_state(state)
    used = torch.empty_like(state)
    with torch.cuda.device(state.device):
        _lib.call("repdl_hip_dropout_next_call", sp, _ptr(used), _stream(state))
    return used


def _pref_logits(logits: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
    """Logits of a preference loss: rows of contiguous elements, any strides between sequences and steps."""
    if not logits.is_cuda:
        raise RuntimeError("logits must be on the GPU (this backend has no CPU path)")
    if logits.dtype not in _DTYPES:
        raise RuntimeError("logits must be float32, bfloat16 or float16, got %s" % logits.dtype)
    if logits.dim() != 3:
        raise RuntimeError("logits must have 3 dimensions (sequence, step, vocabulary), got %d" % logits.dim())
    if logits.shape[0] < 2 or logits.shape[0] % 2:
        raise RuntimeError("logits: the preferred answers, then as many others (got %d sequences)" % logits.shape[0])
    if logits.shape[2] < 1:
        raise RuntimeError("logits: an empty vocabulary")
    if not target.is_cuda or target.dtype != torch.int64:
        raise RuntimeError("target must be int64 on the GPU")
    if tuple(target.shape) != tuple(logits.shape[:2]):
        raise RuntimeError("target must be %s like the logits' rows" % (list(logits.shape[:2]),))
    _same_device(target, logits)
    return logits if logits.stride(2) == 1 or logits.shape[2] == 1 else logits.contiguous()


def preference_loss(logits, target, ref_logps, beta: float, label_smoothing: float, ignore_index: int, grad: bool):
    """Loss, log probabilities of the sequences, and (with ``grad``) row statistics and coefficients for the backward pass."""
    x, t = _pref_logits(logits, target), target.contiguous()
    seqs, steps, vocab = x.shape
    ref = None
    if ref_logps is not None:
        ref = _check(ref_logps, "ref_logps", 1)
        _same_device(ref, x)
        if ref.shape[0] != seqs:
            raise RuntimeError("ref_logps has %d elements for %d sequences" % (ref.shape[0], seqs))
    loss, logps = torch.empty((), dtype=torch.float32, device=x.device), torch.empty((seqs,), dtype=torch.float32, device=x.device)
    stats = torch.empty((seqs, steps, 2), dtype=torch.float32, device=x.device) if grad else None
    coef = torch.empty((seqs,), dtype=torch.float32, device=x.device) if grad else None
    with torch.cuda.device(x.device):
        work, wp, wn = _scratch("repdl_hip_preference_loss_workspace_bytes", x, seqs // 2, steps, vocab)
        _lib.call("repdl_hip_preference_loss_ws", _ptr(x), _ptr(t), _opt(ref), _ptr(loss), _ptr(logps), _opt(stats), _opt(coef), seqs // 2,
                  steps, vocab, x.stride(0), x.stride(1), beta, label_smoothing, ignore_index, _DTYPES[x.dtype], wp, wn, _stream(x))
    return loss, logps, stats, coef


def preference_loss_grad(logits, target, row_stats, coef, grad_loss, ignore_index: int) -> torch.Tensor:
    x, t = _pref_logits(logits, target), target.contiguous()
    seqs, steps, vocab = x.shape
    st, c, g = _check(row_stats, "row_stats", 3), _check(coef, "coef", 1), _check(grad_loss, "grad_loss", 0)
    if tuple(st.shape) != (seqs, steps, 2) or c.shape[0] != seqs:
        raise RuntimeError("row_stats and coef are not those of these logits")
    for v in (st, c, g):
        _same_device(v, x)
    out = torch.empty((seqs, steps, vocab), dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        _lib.call("repdl_hip_preference_loss_grad", _ptr(x), _ptr(t), _ptr(st), _ptr(c), _ptr(g), _ptr(out), seqs // 2, steps, vocab,
                  x.stride(0), x.stride(1), ignore_index, _DTYPES[x.dtype], _stream(x))
    return out


# ---- autograd: the differentiable forms, as csrc/bind.cpp has them ----


class _Once(torch.autograd.Function):
    """The gradients as they are; differentiating them again is an error."""

    @staticmethod
    def forward(ctx, *grads):
        return tuple(None if g is None else g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("this function can be differentiated only once")


def _once(backward):
    """Backward functions whose gradients are not differentiable: where the backward pass is recorded, differentiating them
    again is an error, not a silent zero."""

    @functools.wraps(backward)
    def wrapped(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        return _Once.apply(*(None if g is None else g.detach().requires_grad_() for g in out))

    return wrapped


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, n, weight, bias, eps):
        y, mean, rstd = layer_norm(x, n, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias if weight is None else None, mean, rstd)  # (a bias alone: for its type)
        ctx.n, ctx.shape = n, None if weight is None and bias is None else (bias if weight is None else weight).shape
        return y

    @staticmethod
    @_once
    def backward(ctx, gy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        need_x, _, need_w, need_b = ctx.needs_input_grad[:4]
        gx, gw, gb = layer_norm_grad(gy, x, mean, rstd, ctx.n, weight, bias, need_x, need_w, need_b)
        return gx, None, gw.view(ctx.shape) if need_w else None, gb.view(ctx.shape) if need_b else None, None


def layer_norm_autograd(input, n: int, weight, bias, eps: float) -> torch.Tensor:
    return _LayerNorm.apply(input, n, weight, bias, eps)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, state, seed, call):
        ctx.save_for_backward(state)
        ctx.rest = p, seed, call
        return dropout(x, residual, p, state, seed, call)

    @staticmethod
    @_once
    def backward(ctx, gy):
        p, seed, call = ctx.rest
        # the mask again, from the same call of the generator
        gx = dropout(gy, None, p, ctx.saved_tensors[0], seed, call) if ctx.needs_input_grad[0] else None
        return gx, gy if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout_autograd(input, residual, p: float, state, seed: int, call: int) -> torch.Tensor:
    return _Dropout.apply(input, residual, p, state, seed, call)


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, ref_logps, beta, label_smoothing, ignore_index):
        loss, logps, row_stats, coef = preference_loss(logits, target, ref_logps, beta, label_smoothing, ignore_index, True)
        ctx.save_for_backward(logits, target, row_stats, coef)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(logps)
        ctx.set_materialize_grads(False)
        return loss, logps

    @staticmethod
    @_once
    def backward(ctx, g, _):
        if g is None:
            return (None,) * 6
        logits, target, row_stats, coef = ctx.saved_tensors
        return (preference_loss_grad(logits, target, row_stats, coef, g, ctx.ignore_index),) + (None,) * 5


def preference_loss_autograd(logits, target, ref_logps, beta: float, label_smoothing: float, ignore_index: int):
    return _Preference.apply(logits, target, ref_logps, beta, label_smoothing, ignore_index)
