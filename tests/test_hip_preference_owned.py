"""The preference loss on rows that one token owns: its probability is 1, its log probability 0 (never above), its gradient 0, whatever
the logits' level, type and vocabulary; and rows that it nearly owns."""
import math

import pytest
import torch

import gen
from test_hip_preference import TYPES, reference

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
VOCABS = [2, 50, 1000, 3000, 20000, 50257]
COUNT = 64  # rows: two pairs of 16 steps


def owned(vocab, kind, below):
    """Logits whose rows have their target's logit somewhere in [-40, 40] and all others `below` it."""
    m = (gen.uniform_pm1(1, 4, 16, 1) * 40).to(TYPES[kind])
    t = gen.labels(2, COUNT, vocab).view(4, 16)
    t[0, 0], t[0, 1] = 0, vocab - 1
    x = (m.float() - below).expand(4, 16, vocab).to(TYPES[kind]).contiguous()
    x.scatter_(2, t.unsqueeze(2), m)
    return x.cuda(), t.cuda()


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("vocab", VOCABS)
def test_the_only_possible_token(vocab, kind):
    from repdl_amd.nn import functional as F

    for below in (40.0, math.inf):  # (131072 exp(-40) is far below half a step of 1)
        x, t = owned(vocab, kind, below)
        x.requires_grad_()
        loss, logps = F.preference_loss(x, t, None, 0.3, 0.1)
        (g,) = torch.autograd.grad(loss, x)
        assert not logps.any() and abs(float(loss.detach()) - math.log(2)) <= 2 * U * math.log(2)
        assert not g.gather(2, t.unsqueeze(2)).any()
        others = g.scatter(2, t.unsqueeze(2), 0.0)
        assert others.double().abs().max() <= 0.3 * 1.01 * math.exp(-39) and (below == 40.0 or not others.any())


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("vocab", VOCABS)
def test_a_token_that_is_nearly_certain(vocab, kind):
    """One other token at 4 to 24 below it: 1 - p from 0.02 to 4e-11."""
    from repdl_amd import ops

    x, t = owned(vocab, kind, math.inf)
    far = torch.linspace(4, 24, COUNT, device="cuda").view(4, 16, 1)
    other = (t + 1) % vocab
    value = (x.gather(2, t.unsqueeze(2)).float() - far).to(x.dtype)
    x.scatter_(2, other.unsqueeze(2), value)
    for row in range(COUNT // 4):  # (a sequence of one token: its log probability alone)
        part, target = x[:, row:row + 1], t[:, row:row + 1]
        loss, logps, stats, coef = ops.preference_loss(part, target, None, 0.3)
        want = reference(torch.where(part.isinf(), torch.finfo(x.dtype).min, part), target, None, 0.3, 0.0)[1]
        assert (logps <= 0).all()
        # the two terms: 8.2 U (16 bits) or 2 U, and 0.23 U for each unit of their distance weighted with the term (below 0.1 altogether);
        # the two terms' sum, its factor and the reciprocal: 4 U; the result: half a step of it
        assert ((logps.double().cpu() - want).abs() <= 14.3 * U + want.abs() * U).all()
        g = ops.preference_loss_grad(part, target, stats, coef, torch.ones((), device="cuda"))
        at = g.gather(2, target.unsqueeze(2)).double().flatten()
        assert (at * coef.double().sign() >= 0).all()  # 1 - p is not negative
