"""``torch.nn`` modules whose forward and backward passes use the reproducible
operators -- the counterpart of RepDL's ``repdl/nn/{linear,conv,loss,batchnorm}.py``
module classes.  Each subclasses the PyTorch module it replaces, so parameters,
initialisation and ``state_dict`` layout are PyTorch's.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import ops
from . import functional as F


class Linear(torch.nn.Linear):
    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return F.linear(input, self.weight, self.bias)


class Conv2d(torch.nn.Conv2d):
    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return F.conv2d(input, self.weight, self.bias, self.stride, self.padding, self.dilation, self.groups)


class CrossEntropyLoss(torch.nn.CrossEntropyLoss):
    def forward(self, input: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
        return F.cross_entropy(input, target, weight=self.weight, ignore_index=self.ignore_index,
                               reduction=self.reduction, label_smoothing=self.label_smoothing)


class _BatchNorm(torch.nn.modules.batchnorm._BatchNorm):
    """Batch statistics in training (or when no running statistics are tracked),
    running statistics otherwise (reference batchnorm.py:100-126)."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        self._check_input_dim(input)
        factor = 0.0 if self.momentum is None else self.momentum
        if self.training and self.track_running_stats and self.num_batches_tracked is not None:
            self.num_batches_tracked = self.num_batches_tracked + 1
            if self.momentum is None:
                factor = 1.0 / float(self.num_batches_tracked)
        use_batch = self.training or not self.track_running_stats
        return F.batch_norm(input, self.running_mean, self.running_var, self.weight, self.bias, use_batch,
                            factor, self.eps)


class BatchNorm1d(_BatchNorm):
    _check_input_dim = torch.nn.BatchNorm1d._check_input_dim


class BatchNorm2d(_BatchNorm):
    _check_input_dim = torch.nn.BatchNorm2d._check_input_dim


class LayerNorm(torch.nn.LayerNorm):
    """Layer normalisation whose rows give the same bits in every batch (no counterpart in the reference)."""

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return F.layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)


class Dropout(torch.nn.Dropout):
    """Dropout whose masks are a function of the layer's seed and of how often it has been called, on any device.

    ``rng_state`` (int64: seed, number of the next call) moves with the module and, like everything of ``torch.nn.Dropout``,
    is not part of the state_dict: save it beside the weights to go on with the masks of an interrupted run.  It is no
    buffer: what keeps buffers alike over the ranks of a data-parallel run (DistributedDataParallel's default) would give
    every rank the masks of the first.  Ranks that are to differ take seeds of their own.
    ``seed`` (in [0, 2^63)) defaults to a draw from PyTorch's CPU generator.  A layer that is copied (``copy.deepcopy``)
    draws the same masks as its original: give copies that are to differ a seed of their own.  The call number goes up on
    the device: calls of one layer on several streams at once need an order between them.
    Recomputing a forward pass (activation checkpointing) takes another call and so another mask: use
    ``functional.dropout`` with the state of the first one there.
    ``forward(input, residual)`` adds the residual in the same pass."""

    def __init__(self, p: float = 0.5, inplace: bool = False, seed: Optional[int] = None) -> None:
        super().__init__(p, inplace)
        if inplace:
            raise NotImplementedError("Dropout: in-place is not supported")
        if seed is None:
            seed = int(torch.randint(0, 2 ** 63 - 1, (), dtype=torch.int64, device="cpu"))
        if not 0 <= seed < 2 ** 63:
            raise ValueError("Dropout: the seed is an integer in [0, 2^63)")
        self.rng_state = torch.tensor([seed, 0], dtype=torch.int64)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self.rng_state = fn(self.rng_state)
        return self

    def forward(self, input: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return F.dropout(input, self.p, (0, 0), False, residual)
        return F.dropout(input, self.p, ops.dropout_next_call(self.rng_state), True, residual)


class PreferenceLoss(torch.nn.Module):
    """``functional.preference_loss`` with its settings: (logits, target, ref_logps) -> (loss, log probabilities)."""

    def __init__(self, beta: float = 0.1, label_smoothing: float = 0.0, ignore_index: int = -100) -> None:
        super().__init__()
        self.beta, self.label_smoothing, self.ignore_index = beta, label_smoothing, ignore_index

    def forward(self, logits: torch.Tensor, target: torch.Tensor,
                ref_logps: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        return F.preference_loss(logits, target, ref_logps, self.beta, self.label_smoothing, self.ignore_index)
