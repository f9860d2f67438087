"""Reproducible operators -- the API of RepDL's ``repdl/ops.py:12-157`` served by
the MI355X backend.

Same names, argument order and meaning as the reference.  The reference picks
``backend.cuda`` or ``backend.cpu`` from ``tensor.is_cuda``; here every operator
goes to ``repdl_amd.backend.hip`` and a tensor that is not on the GPU is an
error -- there is no CPU implementation in this package.  ``div`` and ``sqrt``,
which the reference composes from PyTorch calls (``ops.py:98-103, 122-123``), are
HIP kernels with the same IEEE results.  ``exp``, ``log`` (the reference's
internal ``exp2d`` / ``log1d``, ``backend/cpu/math.cpp:14-47``) and ``sum`` are
added as public operators.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from .backend import hip as _hip


def _backend(t: torch.Tensor):
    """The backend module that serves tensor ``t``."""
    if not t.is_cuda:
        raise RuntimeError(
            "repdl_amd.ops: tensor is on %s; this package only implements the GPU (HIP) backend" % t.device
        )
    return _hip


def mm(input: torch.Tensor, mat2: torch.Tensor, transA: bool = False, transB: bool = False) -> torch.Tensor:
    return _backend(input).mm(input, mat2, transA, transB)


def mm_bias(input: torch.Tensor, mat2: torch.Tensor, bias: Optional[torch.Tensor], transA: bool = False,
            transB: bool = False) -> torch.Tensor:
    """``mm(...)`` followed by ``+= bias`` over the rows (the reference's linear layer,
    nn/linear.py:21-22), the one rounded addition made where the chain ends instead of in a
    second pass.  Not in the reference's ``ops``."""
    return _backend(input).mm_bias(input, mat2, bias, transA, transB)


def conv2d(input: torch.Tensor, weight: torch.Tensor, stride: Sequence[int], padding: Sequence[int],
           groups: int) -> torch.Tensor:
    sh, sw = stride
    ph, pw = padding
    return _backend(input).conv2d(input, weight, sh, sw, ph, pw, groups)


def conv2d_bias(input: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], stride: Sequence[int],
                padding: Sequence[int], groups: int) -> torch.Tensor:
    """``conv2d(...)`` followed by ``+= bias`` per output channel (nn/conv.py:27-28), the
    addition made in the kernel's epilogue.  Not in the reference's ``ops``."""
    sh, sw = stride
    ph, pw = padding
    return _backend(input).conv2d_bias(input, weight, bias, sh, sw, ph, pw, groups)


def conv2d_grad_input(input_shape: Sequence[int], weight: torch.Tensor, grad_output: torch.Tensor,
                      stride: Sequence[int], padding: Sequence[int]) -> torch.Tensor:
    # the backend takes grad_output first and only H, W of the input shape
    # (reference ops.py:36-46)
    return _backend(grad_output).conv2d_grad_input(
        grad_output, weight, input_shape[2], input_shape[3], stride[0], stride[1], padding[0], padding[1])


def conv2d_grad_kernel(input: torch.Tensor, weight_shape: Sequence[int], grad_output: torch.Tensor,
                       stride: Sequence[int], padding: Sequence[int]) -> torch.Tensor:
    return _backend(input).conv2d_grad_kernel(
        grad_output, input, weight_shape[2], weight_shape[3], stride[0], stride[1], padding[0], padding[1])


def cross_entropy(input: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
    return _backend(input).cross_entropy(input, target)


def softmax(input: torch.Tensor) -> torch.Tensor:
    return _backend(input).softmax(input)


def div(input: torch.Tensor, other: Union[torch.Tensor, float]) -> torch.Tensor:
    """True IEEE division.  A Python number is rounded to float32 first, exactly
    as the reference's 0-dim float32 tensor is (ops.py:103)."""
    be = _backend(input)
    if isinstance(other, torch.Tensor):
        if other.dim() == 0:
            return be.div_scalar(input, float(other.to(torch.float32)))
        return be.div(input, other.to(input.device))
    return be.div_scalar(input, float(other))


def sqrt(input: torch.Tensor) -> torch.Tensor:
    return _backend(input).sqrt(input)


def exp(input: torch.Tensor) -> torch.Tensor:
    return _backend(input).exp(input)


def log(input: torch.Tensor) -> torch.Tensor:
    return _backend(input).log(input)


def sum1d(input: torch.Tensor, average: bool = False) -> torch.Tensor:
    return _backend(input).sum1d(input, average)


def sum2d_dim0(input: torch.Tensor, keepdim: bool = False, average: bool = False) -> torch.Tensor:
    return _backend(input).sum2d_dim0(input, keepdim, average)


def sum2d_dim1(input: torch.Tensor, keepdim: bool = False, average: bool = False) -> torch.Tensor:
    return _backend(input).sum2d_dim1(input, keepdim, average)


def sum4d_dim023(input: torch.Tensor, keepdim: bool = False, average: bool = False) -> torch.Tensor:
    return _backend(input).sum4d_dim023(input, keepdim, average)


def sum(input: torch.Tensor, dim=None, keepdim: bool = False, average: bool = False) -> torch.Tensor:
    """Sequential-order sum: picks the reference operator that matches the shape.

    1-D (dim None or 0) -> sum1d; 2-D with dim 0 / 1 (or -1) -> sum2d_dim0 / sum2d_dim1;
    4-D with dim (0, 2, 3) -> sum4d_dim023."""
    nd = input.dim()
    if nd == 1 and dim in (None, 0, -1, (0,)):
        return sum1d(input, average)
    if nd == 2 and dim in (0, -2, (0,)):
        return sum2d_dim0(input, keepdim, average)
    if nd == 2 and dim in (1, -1, (1,)):
        return sum2d_dim1(input, keepdim, average)
    if nd == 4 and dim is not None and tuple(dim) == (0, 2, 3):
        return sum4d_dim023(input, keepdim, average)
    raise NotImplementedError("sum over dim=%r of a %d-D tensor has no reproducible operator" % (dim, nd))


def bn_apply(input: torch.Tensor, mean: torch.Tensor, std: torch.Tensor, weight: torch.Tensor,
             bias: torch.Tensor) -> torch.Tensor:
    """``((input - mean) / std) * weight + bias`` with the per-channel vectors broadcast over a
    [N,C,H,W] or [B,F] input: the four rounded operations of the reference's forward
    (nn/batchnorm.py:25-32) in one pass.  Not in the reference's ``ops``."""
    return _backend(input).bn_apply(input, mean, std, weight, bias)


def bn_gvar_term(grad_output: torch.Tensor, input: torch.Tensor, mean: torch.Tensor, coef: torch.Tensor) -> torch.Tensor:
    """``(grad_output * (mean - input)) * coef``: the tensor that grad_var sums (nn/batchnorm.py:56-58)."""
    return _backend(input).bn_gvar_term(grad_output, input, mean, coef)


def bn_gweight_term(input: torch.Tensor, mean: torch.Tensor, std: torch.Tensor, grad_output: torch.Tensor) -> torch.Tensor:
    """``((input - mean) / std) * grad_output``: the tensor that grad_weight sums (nn/batchnorm.py:60-61)."""
    return _backend(input).bn_gweight_term(input, mean, std, grad_output)


def layer_norm(input: torch.Tensor, normalized_shape: Sequence[int], weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               stats: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """The trailing dimensions ``normalized_shape`` normalised: ``(x - mean) * rstd * weight + bias``, every operation
    rounded once in binary32, ``rstd`` the reciprocal of the square root of the biased variance plus eps.  float32,
    bfloat16 or float16; weight and bias of that type or float32.  Returns the output and the rows' mean and rstd
    (float32; None without ``stats``).  Not in the reference's ``ops``."""
    return _backend(input).layer_norm(input, _row_length(input, normalized_shape, weight, bias), weight, bias, eps, stats)


def layer_norm_grad(grad_output: torch.Tensor, input: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                    normalized_shape: Sequence[int], weight: Optional[torch.Tensor] = None, param_like: Optional[torch.Tensor] = None,
                    need_input: bool = True, need_weight: bool = True, need_bias: bool = True):
    """The gradients of ``layer_norm`` with respect to input, weight and bias (None where not needed), from the mean and
    rstd it returned.  Those of weight and bias have ``normalized_shape`` and the type of weight (or of ``param_like`` where
    there is a bias alone; float32 without either); they are sums over all rows in a fixed order."""
    n = _row_length(input, normalized_shape, weight, param_like)
    gx, gw, gb = _backend(input).layer_norm_grad(grad_output, input, mean, rstd, n, weight, param_like, need_input, need_weight, need_bias)
    shape = tuple(normalized_shape)
    return gx, gw if gw is None else gw.view(shape), gb if gb is None else gb.view(shape)


def _row_length(input: torch.Tensor, normalized_shape: Sequence[int], *params: Optional[torch.Tensor]) -> int:
    shape = tuple(normalized_shape)
    if len(shape) == 0 or len(shape) > input.dim() or tuple(input.shape[input.dim() - len(shape):]) != shape:
        raise RuntimeError("layer_norm: the input's shape %s does not end in normalized_shape %s" % (tuple(input.shape), shape))
    n = 1
    for d in shape:
        n *= d
    for p in params:
        if p is not None and tuple(p.shape) != shape:
            raise RuntimeError("layer_norm: a weight or bias of shape %s for normalized_shape %s" % (tuple(p.shape), shape))
    return n


def dropout(input: torch.Tensor, p: float, state: Union[torch.Tensor, Tuple[int, int]],
            residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``input`` with each element dropped with probability p (rounded to a multiple of 2^-32) and the others scaled by
    1 / (1 - p); with ``residual``, that plus residual in the same pass.  Which elements are dropped is a function of
    ``state`` = (seed, call) and their position alone: word j % 4 of Philox4x32-10 at counter (j / 4, call) under the key
    seed decides on element j of the contiguous tensor.  state: an int64 tensor of two elements on the input's device
    (read when the kernel runs, so a captured graph follows it), or two Python integers in [0, 2^64).  The gradient
    with respect to input is the same call on the incoming gradient.  Not in the reference's ``ops``."""
    return _backend(input).dropout(input, residual, float(p), *_dropout_state(state))


def _dropout_state(state: Union[torch.Tensor, Tuple[int, int]]) -> Tuple[Optional[torch.Tensor], int, int]:
    """(tensor, 0, 0) or (None, seed, call), as the backend takes it."""
    if isinstance(state, torch.Tensor):
        return state, 0, 0
    if not isinstance(state, (tuple, list)) or len(state) != 2:
        raise TypeError("dropout: the state is an int64 tensor (seed, call) or two integers, got %r" % (state,))
    seed, call = (int(v) for v in state)
    if not (0 <= seed < 2 ** 64 and 0 <= call < 2 ** 64):
        raise ValueError("dropout: seed and call are integers in [0, 2^64)")
    return None, seed, call


def dropout_next_call(state: torch.Tensor) -> torch.Tensor:
    """A copy of the state (seed, call) of ``dropout``; ``state`` itself goes on to the next call.  One launch, on the
    device: a graph that captures it draws a new mask at every replay."""
    used = _backend(state).dropout_next_call(state)
    torch.autograd.graph.increment_version(state)  # (a backward pass that still needs the old value says so)
    return used


def preference_loss(logits: torch.Tensor, target: torch.Tensor, ref_logps: Optional[torch.Tensor] = None, beta: float = 0.1,
                    label_smoothing: float = 0.0, ignore_index: int = -100, grad: bool = True):
    """Preference loss of pairs of answers from token logits.

    logits [2 P, steps, vocab] (float32, bfloat16, float16; any strides between rows): sequences 0 .. P-1 are the preferred
    answers, P .. 2P-1 the others.  target [2 P, steps] int64: the token each row predicts, ``ignore_index`` where the row is
    not counted.  ref_logps [2 P] float32: the reference model's log probabilities (None: zeros).  With L the summed log
    probabilities and z = beta * ((L_preferred - L_other) - (ref_preferred - ref_other)), the loss is the mean over pairs of
    ``(1 - label_smoothing) * softplus(-z) + label_smoothing * softplus(z)``.
    Returns (loss, L, row_stats, coef); the last two (None without ``grad``) are what ``preference_loss_grad`` takes.
    Not in the reference's ``ops``."""
    return _backend(logits).preference_loss(logits, target, ref_logps, *_preference_settings(beta, label_smoothing, ignore_index), bool(grad))


def _preference_settings(beta: float, label_smoothing: float, ignore_index: int) -> Tuple[float, float, int]:
    if not beta >= 0.0 or not 0.0 <= label_smoothing < 1.0:
        raise ValueError("preference_loss: beta must not be negative and label_smoothing lies in [0, 1)")
    return float(beta), float(label_smoothing), int(ignore_index)


def preference_loss_grad(logits: torch.Tensor, target: torch.Tensor, row_stats: torch.Tensor, coef: torch.Tensor,
                         grad_loss: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """``grad_loss`` (0-dim) times the gradient of ``preference_loss`` with respect to the logits, contiguous, in their type."""
    return _backend(logits).preference_loss_grad(logits, target, row_stats, coef, grad_loss, int(ignore_index))
