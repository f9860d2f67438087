"""Dropout takes the same residuals outside training, and with p = 0, as in training."""
import pytest
import torch

import repdl_amd
from repdl_amd.nn import functional as F

BAD = [lambda x: x[:1], lambda x: x[0], lambda x: x.unsqueeze(0), lambda x: x.float(), lambda x: x.half()]


def check(device):
    x = torch.ones(3, 4, dtype=torch.bfloat16, device=device)
    layer = repdl_amd.nn.Dropout(0.5, seed=1).to(device).eval()
    calls = [lambda r: F.dropout(x, 0.5, (1, 2), training=False, residual=r), lambda r: F.dropout(x, 0.0, (1, 2), residual=r), lambda r: layer(x, r)]
    if device == "cuda":
        calls.append(lambda r: F.dropout(x, 0.5, (1, 2), residual=r))
    for call in calls:
        for bad in BAD:
            with pytest.raises(RuntimeError, match="differ in shape or type"):
                call(bad(x))
        out = call(x)
        assert out.shape == x.shape and out.dtype == x.dtype
    assert torch.equal(calls[0](x), 2 * x)


def test_residuals_outside_training():
    check("cpu")


@pytest.mark.gpu
def test_residuals_in_every_mode():
    check("cuda")
