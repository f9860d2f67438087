"""Reproducible ``torch.nn`` layers (RepDL ``repdl/nn/__init__.py:4-8``), and LayerNorm, Dropout and PreferenceLoss in the same manner."""
from . import functional
from .modules import BatchNorm1d, BatchNorm2d, Conv2d, CrossEntropyLoss, Dropout, LayerNorm, Linear, PreferenceLoss

__all__ = ["functional", "BatchNorm1d", "BatchNorm2d", "Conv2d", "CrossEntropyLoss", "Dropout", "LayerNorm", "Linear", "PreferenceLoss"]
