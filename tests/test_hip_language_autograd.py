"""The differentiable forms of layer norm, dropout and the preference loss: the compiled binding's and the ctypes binding's give the
same gradients, only the wanted ones are made, a second derivative and a changed input are errors, and two backward passes at once do not
meet."""
import threading

import pytest
import torch

import gen

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["ext", "ctypes"])
def binding(request):
    from repdl_amd.backend import hip

    before = hip.BINDING
    if request.param == "ext" and before != "ext":
        pytest.skip("the compiled binding has not been built")
    hip.use_binding(request.param)
    yield request.param
    hip.use_binding(before)


def _inputs():
    x = gen.normal_like(1, 6, 40).cuda()
    w, b = gen.normal_like(2, 40).cuda(), gen.normal_like(3, 40).cuda()
    t = gen.labels(4, 6, 40).view(2, 3).cuda()
    return x, w, b, t


@pytest.mark.parametrize("wanted", range(1, 8))
def test_only_the_wanted_gradients(binding, wanted):
    from repdl_amd import ops
    from repdl_amd.nn import functional as F

    x, w, b, _ = _inputs()
    for i, t in enumerate((x, w, b)):
        t.requires_grad_(bool(wanted >> i & 1))
    gy = gen.normal_like(5, 6, 40).cuda()
    y = F.layer_norm(x, 40, w, b)
    y.backward(gy)
    _, mean, rstd = ops.layer_norm(x, (40,), w, b)
    for t, g in zip((x, w, b), ops.layer_norm_grad(gy, x, mean, rstd, (40,), w)):
        assert (t.grad is not None) == t.requires_grad and (t.grad is None or torch.equal(t.grad, g))


def test_a_bias_alone(binding):
    from repdl_amd.nn import functional as F

    x = gen.normal_like(8, 6, 4, 10).to(torch.bfloat16).cuda()
    b = gen.normal_like(9, 4, 10).to(torch.bfloat16).cuda().requires_grad_()
    gy = gen.normal_like(10, 6, 4, 10).to(torch.bfloat16).cuda()
    F.layer_norm(x, (4, 10), None, b).backward(gy)
    assert b.grad.shape == b.shape and b.grad.dtype == b.dtype
    # (six terms: at most 6 + 48 roundings of the sum of magnitudes, and the one to bfloat16)
    want = gy.double().sum(0)
    assert ((b.grad.double() - want).abs() <= gy.double().abs().sum(0) * 54 * 2.0 ** -24 + want.abs() * 2.0 ** -8).all()


def test_residual_of_dropout_alone(binding):
    from repdl_amd.nn import functional as F

    x, r = gen.normal_like(6, 50).cuda(), gen.normal_like(7, 50).cuda().requires_grad_()
    for state in ((1, 2), torch.tensor([1, 2], device="cuda")):
        r.grad = None
        F.dropout(x, 0.5, state, residual=r).sum().backward()
        assert torch.equal(r.grad, torch.ones_like(r))
        assert not F.dropout(x, 0.5, state, residual=r.detach()).requires_grad


def test_a_second_derivative_is_refused(binding):
    from repdl_amd.nn import functional as F

    x, w, b, t = _inputs()
    x.requires_grad_()
    outs = [lambda: F.layer_norm(x, 40, w, b).square().sum(), lambda: F.dropout(x, 0.5, (1, 2)).square().sum(),
            lambda: F.preference_loss(x.view(2, 3, 40), t)[0].square(),
            lambda: F.preference_loss(x.view(2, 3, 40), t)[0], lambda: F.layer_norm(x, 40, w, b).sum(), lambda: F.dropout(x, 0.5, (1, 2)).sum()]
    for f in outs:
        (g,) = torch.autograd.grad(f(), x)
        (h,) = torch.autograd.grad(f(), x, create_graph=True)  # (the first derivative of a recorded backward pass is there)
        assert torch.equal(g, h.detach()) and h.requires_grad
        with pytest.raises(RuntimeError, match="only once"):
            (x.sum() + h.square().sum()).backward()  # (a penalty on the gradient, beside a term that has one)


def test_a_changed_input_is_noticed(binding):
    from repdl_amd.nn import functional as F

    x, w, b, t = _inputs()
    leaf = x.clone().requires_grad_()
    for f in (lambda v: F.layer_norm(v, 40, w, b), lambda v: F.preference_loss(v.view(2, 3, 40), t)[0]):
        v = leaf * 1.0
        y = f(v)
        v.add_(1.0)
        with pytest.raises(RuntimeError):
            y.sum().backward()


def test_unused_loss_and_two_uses(binding):
    from repdl_amd.nn import functional as F

    x, w, b, t = _inputs()
    x.requires_grad_()
    loss, logps = F.preference_loss(x.view(2, 3, 40), t)
    assert loss.requires_grad and not logps.requires_grad
    (g,) = torch.autograd.grad(loss, x)
    both = F.preference_loss(x.view(2, 3, 40), t)[0] + F.preference_loss(x.view(2, 3, 40), t)[0]
    assert torch.equal(torch.autograd.grad(both, x)[0], g + g)
    y = F.layer_norm(x, 40, w, b)
    (one,) = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    (two,) = torch.autograd.grad(y, x, torch.ones_like(y))  # the graph once more
    assert torch.equal(one, two)
    expanded = torch.autograd.grad(F.layer_norm(x, 40, w, b).sum(), x)[0]  # an incoming gradient of stride 0
    assert torch.equal(expanded, one)


def test_threads_with_streams_of_their_own(binding):
    """Two host threads, each on its own stream: forward and backward of all three, many times, the same bits as alone."""
    from repdl_amd.nn import functional as F

    x, w, b, t = _inputs()

    def step(scale):
        v = (x * scale).requires_grad_()
        h = F.dropout(F.layer_norm(v, 40, w, b), 0.25, (3, 4), residual=v)
        loss = F.preference_loss(h.view(2, 3, 40), t)[0]
        return [loss.detach()] + list(torch.autograd.grad(loss, v))

    want = [step(1.0), step(2.0)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = step(1.0 + i)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(p, q) for p, q in zip(got, want[i])):
                        bad.append(i)
        except Exception as e:  # noqa: BLE001 (reported by the test)
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not bad, bad


def test_a_leaf_of_a_living_eager_graph_is_refused_under_capture():
    """Only forward passes are captured here: the refusal comes before anything that a backward pass could meet."""
    from repdl_amd.backend import hip
    from repdl_amd.nn import functional as F

    if hip.BINDING != "ext":
        pytest.skip("the compiled binding's check")
    x, w, b, t = _inputs()
    calls = {
        "weight": (w, lambda: F.layer_norm(x, (40,), w, b)),
        "input": (x, lambda: F.dropout(x, 0.5, (3, 0))),
        "logits": (None, None),
    }
    logits = x.view(2, 3, 40).clone()
    calls["logits"] = (logits, lambda: F.preference_loss(logits, t)[0])
    for name, (leaf, call) in calls.items():
        leaf.requires_grad_()
        call()  # (the first launch loads the kernels; its graph dies at once)
        eager = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = x.detach() + 1  # (something to capture)
            with pytest.raises(RuntimeError, match=f"{name} still belongs to an eager graph"):
                call()
            with torch.no_grad():
                call()  # (nothing is recorded: no leaf is met)
        torch.autograd.grad(eager.sum(), leaf)
        del eager, held
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            again = call().detach()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, call().detach())
        side = torch.cuda.Stream()  # (an eager graph of a side stream stands in nobody's way)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            again = call().detach()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, eager.detach())
        del eager
        leaf.requires_grad_(False)
