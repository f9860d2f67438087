"""Layer norm, dropout and the preference loss have no forward-mode derivative and say so, as the module's other functions do: a tangent
that is passed by would read as zero.  (The refusal comes before the device is looked at.)"""
import pytest
import torch
from torch.autograd import forward_ad

from repdl_amd.nn import functional as F


def calls(device):
    x, w = torch.randn(4, 8, device=device), torch.randn(8, device=device)
    logits, target = torch.randn(2, 3, 5, device=device), torch.zeros(2, 3, dtype=torch.int64, device=device)
    ref = torch.zeros(2, device=device)
    return [(x, lambda v: F.layer_norm(v, 8, w, w)), (w, lambda v: F.layer_norm(x, 8, v)), (w, lambda v: F.layer_norm(x, 8, None, v)),
            (x, lambda v: F.dropout(v, 0.5, (1, 2))), (x, lambda v: F.dropout(x, 0.5, (1, 2), residual=v)),
            (logits, lambda v: F.preference_loss(v, target)), (ref, lambda v: F.preference_loss(logits, target, v))]


def check(device):
    for at, call in calls(device):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(at, torch.ones_like(at))
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError):
                    call(dual)
            with pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(at.clone().requires_grad_(), torch.ones_like(at)))
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda v: F.layer_norm(v, 8), (torch.randn(4, 8, device=device),), (torch.ones(4, 8, device=device),))
    with forward_ad.dual_level():  # outside training dropout is the identity, which has its tangent
        dual = forward_ad.make_dual(torch.ones(4, device=device), torch.full((4,), 3.0, device=device))
        assert forward_ad.unpack_dual(F.dropout(dual, 0.5, (1, 2), training=False, residual=dual)).tangent.tolist() == [6.0] * 4


def test_tangents_are_refused():
    check("cpu")


@pytest.mark.gpu
def test_tangents_are_refused_on_the_gpu():
    check("cuda")
    for at, call in calls("cuda"):  # a level without tangents is no obstacle
        with forward_ad.dual_level():
            call(at)
