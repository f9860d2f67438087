"""Dropout on the GPU: the mask against Philox in numpy, bit for bit; values in every type; the residual form; the gradient;
the state on the device; streams, graphs, refusals."""
import numpy as np
import pytest
import torch

import gen
import philox

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def expected(x, p, seed, call, residual=None, first=0):
    """The definition with its roundings: one product in binary32, one sum in binary32, one rounding to the type."""
    keep = torch.from_numpy(philox.words(x.numel(), seed, call, first).astype(np.int64)).view(x.shape) >= round(p * 2 ** 32)
    scaled = x.float() * torch.tensor(1 / (1 - p), dtype=torch.float32) if p < 1 else torch.zeros_like(x.float())
    if residual is None:
        return torch.where(keep, scaled, torch.zeros(())).to(x.dtype), keep
    return torch.where(keep, residual.float() + scaled, residual.float()).to(x.dtype), keep


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 255, 1024, 4097, 8191, 65537, 1000003])
def test_mask_and_values(n, kind):
    from repdl_amd import ops

    x, r = gen.normal_like(n, n).to(TYPES[kind]), gen.normal_like(n + 1, n).to(TYPES[kind])
    for p, seed, call in ((0.1, 12345, 0), (0.5, 2 ** 63 + 11, 2 ** 40 + 3), (0.999, 0, 2 ** 64 - 1)):
        want, keep = expected(x, p, seed, call)
        assert torch.equal(ops.dropout(x.cuda(), p, (seed, call)).cpu(), want)
        assert torch.equal(ops.dropout(x.cuda(), p, (seed, call), r.cuda()).cpu(), expected(x, p, seed, call, r)[0])
        if n > 100000:  # six standard deviations of a binomial count
            assert abs(int((~keep).sum()) - n * p) <= 6 * (n * p * (1 - p)) ** 0.5


@pytest.mark.parametrize("n", [8, 4096, 4097, 4099, 4103])
def test_two_roundings_in_float16_everywhere(n):
    """A product whose rounding to binary32 lies half way between two float16 numbers: the second rounding then goes to the even
    one, at the end of a tensor (element by element) as inside (in granules)."""
    from repdl_amd import ops

    p = 0.7500858221038925  # 0.7109375 * float(1 / (1 - p)) rounds to 2.8447265625, half way between 2.84375 and 2.845703125
    x = torch.full((n,), 0.7109375, dtype=torch.float16)
    want, keep = expected(x, p, 3, 4)
    assert keep[-8:].any() and set(want[keep].tolist()) == {2.84375}
    assert torch.equal(ops.dropout(x.cuda(), p, (3, 4)).cpu(), want)
    for at in range(n - 8, n):  # the same element as the last one
        assert torch.equal(ops.dropout(x[:at + 1].cuda(), p, (3, 4)).cpu(), want[:at + 1])


def test_known_answers():
    """Three blocks of the generator from the paper's reference vectors, as masks: word >= round(p 2^32) at thresholds on
    either side of each word."""
    from repdl_amd import ops

    answers = ((0, 0, 0, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),)
    for seed, call, at, text in answers:
        for k, word in enumerate(int(v, 16) for v in text.split()):
            for threshold, kept in ((word, True), (word + 1, False)):
                y = ops.dropout(torch.ones(4, device="cuda"), threshold / 2 ** 32, (seed, call))
                assert bool(y[k]) == kept
    c = philox.block([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF))
    assert [int(v) for v in c] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    c = philox.block([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0))
    assert [int(v) for v in c] == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_types_share_the_mask_and_odd_addresses_do_not_matter():
    from repdl_amd import ops

    n = 10007
    masks = [ops.dropout(torch.ones(n, device="cuda", dtype=t), 0.3, (5, 6)) != 0 for t in TYPES.values()]
    assert torch.equal(masks[0], masks[1]) and torch.equal(masks[0], masks[2])
    for t in TYPES.values():
        x = gen.normal_like(3, n + 1).to(t).cuda()
        assert torch.equal(ops.dropout(x[1:], 0.3, (5, 6)), ops.dropout(x[1:].clone(), 0.3, (5, 6)))
    x = gen.normal_like(4, 100, 50).cuda()
    assert torch.equal(ops.dropout(x.t(), 0.3, (5, 6)), ops.dropout(x.t().contiguous(), 0.3, (5, 6)))  # the positions of the result


def test_limits_of_p_and_special_values():
    from repdl_amd import ops

    x = gen.normal_like(7, 1000).cuda()
    x[::9], x[1::9], x[2::9] = float("inf"), float("nan"), -0.0
    r = gen.normal_like(8, 1000).cuda()
    assert not ops.dropout(x, 1.0, (1, 2)).any()          # dropped infinities and NaN are zeros
    assert torch.equal(ops.dropout(x, 1.0, (1, 2), r), r)
    same = ops.dropout(x, 0.0, (1, 2))
    assert torch.equal(same.view(torch.int32), x.view(torch.int32))
    y, keep = expected(x.cpu(), 0.5, 1, 2)
    got = ops.dropout(x, 0.5, (1, 2)).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(y)) and torch.equal(got[~torch.isnan(y)], y[~torch.isnan(y)])
    assert ops.dropout(x[:0], 0.5, (1, 2)).shape == (0,)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("on_device", [True, False])
def test_gradient(kind, on_device):
    from repdl_amd import ops
    from repdl_amd.nn import functional as F

    t = TYPES[kind]
    seed, call = 99, 7
    state = torch.tensor([seed, call], device="cuda") if on_device else (seed, call)
    x, r, gy = (gen.normal_like(20 + i, 33, 129).to(t).cuda() for i in range(3))
    x.requires_grad_()
    r.requires_grad_()
    y = F.dropout(x, 0.2, state, residual=r)
    assert torch.equal(y.detach().cpu(), expected(x.detach().cpu(), 0.2, seed, call, r.detach().cpu())[0])
    gx, gr = torch.autograd.grad(y, (x, r), gy)
    assert torch.equal(gx.cpu(), expected(gy.cpu(), 0.2, seed, call)[0]) and torch.equal(gr, gy)
    (gx,) = torch.autograd.grad(F.dropout(x, 0.2, state), x, gy.t().contiguous().t())  # a gradient of other strides
    assert torch.equal(gx.cpu(), expected(gy.cpu(), 0.2, seed, call)[0])
    assert F.dropout(x, 0.2, state, training=False) is x
    assert torch.equal(F.dropout(x, 0.0, state, residual=r), r + x)
    if kind == "f32":  # against differences: small whole numbers, whose sums are exact, in a function that is linear in x
        u, v = gen.small_ints(30, 33, 129).cuda(), gen.small_ints(31, 33, 129).cuda()
        slope = ops.dropout(u + v, 0.5, state) - ops.dropout(u, 0.5, state)
        (gx,) = torch.autograd.grad(F.dropout(x, 0.5, state), x, torch.ones_like(x))
        assert torch.equal(slope, gx * v)


def test_state_on_the_device():
    from repdl_amd import ops
    from repdl_amd.nn import functional as F

    state = torch.tensor([2 ** 62 + 5, 2 ** 32 - 1], device="cuda")
    used = ops.dropout_next_call(state)
    assert used.tolist() == [2 ** 62 + 5, 2 ** 32 - 1] and state.tolist() == [2 ** 62 + 5, 2 ** 32]
    x = gen.normal_like(40, 5000).cuda()
    assert torch.equal(ops.dropout(x, 0.4, used), ops.dropout(x, 0.4, (2 ** 62 + 5, 2 ** 32 - 1)))
    # negative numbers are the upper half of the unsigned range
    assert torch.equal(ops.dropout(x, 0.4, torch.tensor([-1, -2], device="cuda")), ops.dropout(x, 0.4, (2 ** 64 - 1, 2 ** 64 - 2)))
    # a state that went on before the backward pass is noticed
    x.requires_grad_()
    y = F.dropout(x, 0.4, state)
    ops.dropout_next_call(state)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_module():
    import repdl_amd

    m = repdl_amd.nn.Dropout(0.25, seed=77).cuda()
    assert list(m.state_dict()) == list(torch.nn.Dropout().state_dict())
    x = gen.normal_like(50, 64, 100).cuda()
    for call in range(3):
        assert torch.equal(m(x).cpu(), expected(x.cpu(), 0.25, 77, call)[0])
    assert torch.equal(m(x, x).cpu(), expected(x.cpu(), 0.25, 77, 3, x.cpu())[0])
    m.eval()
    assert m(x) is x and m.rng_state.tolist() == [77, 4]
    torch.manual_seed(3)
    a = repdl_amd.from_torch_module(torch.nn.Sequential(torch.nn.Dropout(0.1), torch.nn.Dropout(0.2)), language_layers=True)
    torch.manual_seed(3)
    b = repdl_amd.from_torch_module(torch.nn.Sequential(torch.nn.Dropout(0.1), torch.nn.Dropout(0.2)), language_layers=True)
    assert [m.p for m in a] == [0.1, 0.2] and torch.equal(a[0].rng_state, b[0].rng_state) and not torch.equal(a[0].rng_state, a[1].rng_state)
    with pytest.raises(NotImplementedError):
        repdl_amd.nn.Dropout(0.1, inplace=True)


def test_graph_draws_a_new_mask_at_every_replay():
    import repdl_amd

    m = repdl_amd.nn.Dropout(0.5, seed=5).cuda()
    x = gen.normal_like(60, 200, 33).cuda().requires_grad_()
    gy = gen.normal_like(61, 200, 33).cuda()
    m(x)  # call 0, before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
        (gx,) = torch.autograd.grad(y, x, gy)
    for call in range(1, 5):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.detach().cpu(), expected(x.detach().cpu(), 0.5, 5, call)[0])
        assert torch.equal(gx.cpu(), expected(gy.cpu(), 0.5, 5, call)[0])
    assert torch.equal(m(x).detach().cpu(), expected(x.detach().cpu(), 0.5, 5, 5)[0])  # and eager calls go on from there


def test_side_stream_and_both_bindings():
    from repdl_amd import ops
    from repdl_amd.backend import hip_ctypes

    x = gen.normal_like(70, 12345).cuda()
    want = ops.dropout(x, 0.3, (1, 1), x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.dropout(x, 0.3, (1, 1), x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert torch.equal(hip_ctypes.dropout(x, x, 0.3, None, 1, 1), want)
    state = torch.tensor([1, 1], device="cuda")
    assert torch.equal(hip_ctypes.dropout(x, x, 0.3, state, 0, 0), want)
    assert hip_ctypes.dropout_next_call(state).tolist() == [1, 1] and state.tolist() == [1, 2]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("residual", [False, True])
def test_large_tensors_have_the_bits_of_their_beginning(kind, residual):
    """256 MB and more are moved past the caches, by other instructions."""
    from repdl_amd import ops

    n = (1 << 28) // torch.finfo(TYPES[kind]).bits * 8 + 77
    x = gen.normal_like(80, 1 << 20).to(TYPES[kind]).cuda().repeat((n >> 20) + 1)[:n]
    r = x.flip(0) if residual else None
    y = ops.dropout(x, 0.3, (8, 9), r)
    m = n // 2 + 3
    assert torch.equal(y[:m], ops.dropout(x[:m], 0.3, (8, 9), r[:m] if residual else None))
    first = (n - 4096) // 4 * 4  # and the end against the definition
    want, _ = expected(x[first:].cpu(), 0.3, 8, 9, r[first:].cpu() if residual else None, first)
    assert torch.equal(y[first:].cpu(), want)


def test_more_elements_than_32_bits_count():
    from repdl_amd import ops

    n = (1 << 32) + 4099                              # (in 16 bits; block numbers past 2^30, element numbers past 2^32)
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = ops.dropout(x, 0.5, (12, 34))
    for first, count in ((0, 1000), ((1 << 31) - 512, 1024), ((1 << 32) - 512, 4611)):
        keep = torch.from_numpy(philox.words(count, 12, 34, first).astype(np.int64)) >= 1 << 31
        assert torch.equal(y[first:first + count].cpu() != 0, keep)


def test_refusals():
    from repdl_amd import ops
    from repdl_amd.nn import functional as F

    x = torch.zeros(8, device="cuda")
    state = torch.tensor([1, 2], device="cuda")
    bad = [lambda: ops.dropout(x.cpu(), 0.5, (1, 2)), lambda: ops.dropout(x.double(), 0.5, (1, 2)), lambda: ops.dropout(x, 1.5, (1, 2)),
           lambda: ops.dropout(x, -0.1, (1, 2)), lambda: ops.dropout(x, float("nan"), (1, 2)), lambda: ops.dropout(x, 0.5, (-1, 2)),
           lambda: ops.dropout(x, 0.5, (1, 2 ** 64)), lambda: ops.dropout(x, 0.5, state.cpu()), lambda: ops.dropout(x, 0.5, state.int()),
           lambda: ops.dropout(x, 0.5, state[:1]), lambda: ops.dropout(x, 0.5, (1, 2), x[:4]), lambda: ops.dropout(x, 0.5, (1, 2), x.half()),
           lambda: F.dropout(x, 1.01, (1, 2)), lambda: ops.dropout_next_call(state.cpu()), lambda: ops.dropout_next_call(x)]
    for call in bad:
        with pytest.raises((RuntimeError, ValueError)):
            call()
    assert state.tolist() == [1, 2]
