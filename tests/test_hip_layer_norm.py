"""Layer normalisation on the GPU: forward and backward against the definition in binary64, at row lengths around every
change of the threads per row, in every type, for rows that are no whole granules and odd addresses; the bits of a row do
not depend on its batch; refusals; streams, graphs and autograd."""
import pytest
import torch

import gen
import norm_model

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
STEP = {t: torch.finfo(t).eps / 2 for t in TYPES.values()}  # half a step of the type, relative
U = 2.0 ** -24


def reference(x, w, b, eps, gy=None):
    """y, gx, gw, gb in binary64"""
    x = x.detach().double().cpu()
    w = torch.ones(x.shape[1], dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(x.shape[1], dtype=torch.float64) if b is None else b.detach().double().cpu()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    y = xh * w + b
    if gy is None:
        return y, xh, rstd
    gy = gy.double().cpu()
    g = gy * w
    gx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return y, xh, rstd, gx, (gy * xh).sum(0), gy.sum(0)


def data(rows, cols, kind, wkind, seed=1):
    x = (gen.normal_like(seed, rows, cols) * 2 + gen.normal_like(seed + 1, rows, 1)).to(kind).cuda()
    w = (1 + 0.25 * gen.normal_like(seed + 2, cols)).to(wkind).cuda()
    b = (0.5 * gen.normal_like(seed + 3, cols)).to(wkind).cuda()
    gy = gen.normal_like(seed + 4, rows, cols).to(kind).cuda()
    return x, w, b, gy


def depth(n):
    """Additions on the longest path of a row's sum (at most 16 elements a thread, log2 of the rest), and one more per wave."""
    return 16 + 6 + 16 + n // 4096


def check_forward(y, x, w, b, eps=1e-5):
    want, xh, rstd = reference(x, w, b, eps)
    n = x.shape[1]
    spread = x.detach().double().cpu().abs().amax(1, keepdim=True)
    # the mean is off by (depth + 2) roundings of at most the row's largest value, each of which the scale rstd carries over
    # to y; the variance's relative error is at most (depth + 6) roundings plus twice the mean's in units of the spread,
    # halved by the root; four roundings follow, and the one to the type
    mean_err = (depth(n) + 2) * U * spread
    tol = (mean_err * rstd * (1 + xh.abs()) + xh.abs() * (depth(n) + 10) * U)
    wa = torch.ones(n, dtype=torch.float64) if w is None else w.detach().double().cpu().abs()
    tol = tol * wa + want.abs() * (2 * U + STEP[y.dtype]) + (xh.abs() * wa) * 2 * U + torch.finfo(y.dtype).smallest_normal
    err = (y.detach().double().cpu() - want).abs()
    assert (err <= tol).all(), (float((err / tol).max()), x.shape, y.dtype)


def check_backward(got, x, w, b, gy, eps=1e-5):
    y, xh, rstd, gx, gw, gb = reference(x, w, b, eps, gy)
    rows, n = x.shape
    spread = x.detach().double().cpu().abs().amax(1, keepdim=True)
    gyd = gy.double().cpu()
    g = (gyd if w is None else gyd * w.detach().double().cpu()).abs()
    xerr = (depth(n) + 2) * U * spread * rstd * (1 + xh.abs()) + xh.abs() * (depth(n) + 10) * U  # of xh, as above
    k = depth(n) + 8
    tol = rstd * (k * U * (g + g.mean(1, keepdim=True) + xh.abs() * (g * xh.abs()).mean(1, keepdim=True))
                  + xerr * (g * xh.abs()).mean(1, keepdim=True) + xh.abs() * (g * xerr).mean(1, keepdim=True))
    tol = tol + gx.abs() * ((depth(n) + 10) * U + mean_rel(x, rstd, n) + STEP[x.dtype]) + torch.finfo(x.dtype).smallest_normal
    if got[0] is not None:
        err = (got[0].double().cpu() - gx).abs()
        assert (err <= tol).all(), (float((err / tol).max()), x.shape, x.dtype)
    # sums over rows: at most rows / 256 (+ the teams of a workgroup) + 64 + 64 additions deep, each off by U of the sum of magnitudes
    # (up to 256 rows: at most 16 rows and 64 sums)
    d = rows // 256 + 64 + 48 + 16
    for t, want, terms, extra in ((got[1], gw, gyd.abs() * xh.abs(), (gyd.abs() * xerr).sum(0)), (got[2], gb, gyd.abs(), 0.0)):
        if t is not None:
            tol = d * U * terms.sum(0) + extra + want.abs() * STEP[t.dtype] + torch.finfo(t.dtype).smallest_normal
            err = (t.double().cpu() - want).abs()
            assert (err <= tol).all(), (float((err / tol).max()), x.shape, t.dtype)


def mean_rel(x, rstd, n):
    """what the mean's error makes of rstd, relative"""
    return (depth(n) + 2) * U * x.detach().double().cpu().abs().amax(1, keepdim=True) * rstd


SHAPES = [(1, 1), (3, 1), (5, 2), (7, 15), (64, 16), (65, 17), (33, 63), (40, 64), (9, 65), (130, 127), (17, 255), (600, 256), (21, 257), (1030, 513),
          (3, 1000), (515, 1024), (1, 1025), (6, 2049), (5, 4096), (4, 4099), (3, 8193), (2, 16384), (2, 16385), (3, 20001), (1, 70001)]


@pytest.mark.parametrize("kind,wkind", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(shape, kind, wkind):
    from repdl_amd.nn import functional as F

    x, w, b, gy = data(*shape, TYPES[kind], TYPES[wkind])
    for t in (x, w, b):
        t.requires_grad_()
    y = F.layer_norm(x, shape[1:], w, b)
    assert y.dtype == x.dtype and y.shape == x.shape
    check_forward(y, x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), gy)
    assert [g.dtype for g in grads] == [t.dtype for t in (x, w, b)]
    check_backward(grads, x, w, b, gy)
    with torch.no_grad():  # the form without statistics: the same bits
        assert torch.equal(F.layer_norm(x, shape[1:], w, b), y)


@pytest.mark.parametrize("which", ["weight", "bias", "none"])
def test_missing_parameters(which):
    from repdl_amd.nn import functional as F

    x, w, b, gy = data(37, 300, torch.bfloat16, torch.float32)
    w, b = (w.requires_grad_() if which == "weight" else None), (b.requires_grad_() if which == "bias" else None)
    x.requires_grad_()
    y = F.layer_norm(x, (300,), w, b)
    check_forward(y, x, w, b)
    wrt = [t for t in (x, w, b) if t is not None]
    grads = dict(zip([id(t) for t in wrt], torch.autograd.grad(y, wrt, gy)))
    check_backward([grads.get(id(t)) if t is not None else None for t in (x, w, b)], x, w, b, gy)
    x.requires_grad_(False)
    if w is not None:  # the weight's gradient alone
        (gw,) = torch.autograd.grad(F.layer_norm(x, (300,), w, b), w, gy)
        check_backward([None, gw, None], x, w, b, gy)


def test_gradients_against_differences():
    """d/dt loss(x + t v) by the difference of two binary64 evaluations of the definition, against the gradient's product
    with v: the gradient's binary32 error is 2^-24 times some tens of roundings of terms of the product's size."""
    from repdl_amd.nn import functional as F

    x, w, b, gy = data(13, 77, torch.float32, torch.float32, seed=40)
    for t in (x, w, b):
        t.requires_grad_()
    grads = torch.autograd.grad(F.layer_norm(x, (77,), w, b), (x, w, b), gy)
    for i, (t, g) in enumerate(zip((x, w, b), grads)):
        v = gen.normal_like(50 + i, *t.shape).double()
        h, vals = 1e-5, []
        for s in (h, -h):
            args = [u.detach().double().cpu() + (s * v if j == i else 0) for j, u in enumerate((x, w, b))]
            vals.append((reference(args[0], args[1], args[2], 1e-5)[0] * gy.double().cpu()).sum())
        want = float((vals[0] - vals[1]) / (2 * h))
        size = float((g.double().cpu() * v).abs().sum())
        # (the difference itself is off by h^2 times the third derivative, 1e-10 of it here, and by 2^-52 of the sum / h)
        assert abs(float((g.double().cpu() * v).sum()) - want) <= size * 100 * U + 1e-6


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [5, 64, 1000, 1100, 1280, 4096, 9000])
def test_rows_do_not_depend_on_their_batch(cols, kind):
    from repdl_amd import ops

    x, w, b, gy = data(300, cols, TYPES[kind], torch.float32, seed=60)
    y, mean, rstd = ops.layer_norm(x, (cols,), w, b)
    gx = ops.layer_norm_grad(gy, x, mean, rstd, (cols,), w)[0]
    for at, n in ((0, 1), (7, 1), (100, 64), (299, 1)):
        part = x[at:at + n].clone()
        yp, mp, rp = ops.layer_norm(part, (cols,), w, b)
        assert torch.equal(yp, y[at:at + n]) and torch.equal(mp, mean[at:at + n]) and torch.equal(rp, rstd[at:at + n])
        assert torch.equal(ops.layer_norm_grad(gy[at:at + n].clone(), part, mp, rp, (cols,), w)[0], gx[at:at + n])
    again = ops.layer_norm_grad(gy, x, mean, rstd, (cols,), w)
    for a, c in zip(again, ops.layer_norm_grad(gy, x, mean, rstd, (cols,), w)):
        assert torch.equal(a, c)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_odd_addresses_and_strides(kind):
    from repdl_amd import ops

    t = TYPES[kind]
    x, w, b, gy = data(9, 131, t, t, seed=70)
    want = ops.layer_norm(x, (131,), w, b)
    grads = ops.layer_norm_grad(gy, x, want[1], want[2], (131,), w)
    shift = lambda v: torch.cat([v.new_zeros(1), v.reshape(-1)])[1:].view(v.shape)  # noqa: E731 (one element off every boundary)
    xs, ws, bs, gs = (shift(v) for v in (x, w, b, gy))
    assert xs.data_ptr() % 16 == x.element_size()
    got = ops.layer_norm(xs, (131,), ws, bs)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert all(torch.equal(p, q) for p, q in zip(ops.layer_norm_grad(gs, xs, got[1], got[2], (131,), ws), grads))
    wide = torch.zeros(9, 200, dtype=t, device="cuda")
    wide[:, 30:161] = x
    assert torch.equal(ops.layer_norm(wide[:, 30:161], (131,), w, b)[0], want[0])
    assert torch.equal(ops.layer_norm(x.t().contiguous().t(), (131,), w, b)[0], want[0])


def test_several_normalized_dimensions_and_module():
    import repdl_amd
    from repdl_amd.nn import functional as F

    x = gen.normal_like(80, 4, 6, 5, 7).cuda()
    w, b = gen.normal_like(81, 5, 7).cuda(), gen.normal_like(82, 5, 7).cuda()
    y = F.layer_norm(x, (5, 7), w, b)
    assert torch.equal(y.reshape(24, 35), F.layer_norm(x.reshape(24, 35), 35, w.reshape(35), b.reshape(35)))
    src = torch.nn.LayerNorm((5, 7), eps=1e-3)
    with torch.no_grad():
        src.weight.copy_(w)
        src.bias.copy_(b)
    m = repdl_amd.from_torch_module(torch.nn.Sequential(src), language_layers=True).cuda()
    assert type(m[0]) is repdl_amd.nn.LayerNorm and m[0].eps == 1e-3
    x.requires_grad_()
    out = m(x)
    assert torch.equal(out, F.layer_norm(x, (5, 7), w, b, 1e-3))
    out.sum().backward()
    assert x.grad.shape == x.shape and m[0].weight.grad.shape == (5, 7) and m[0].bias.grad.shape == (5, 7)
    assert type(repdl_amd.from_torch_module(torch.nn.Sequential(src))[0]) is torch.nn.LayerNorm  # only where asked for


def test_empty_and_special_rows():
    from repdl_amd import ops
    from repdl_amd.nn import functional as F

    w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
    x = torch.zeros(0, 8, device="cuda", requires_grad=True)
    y = F.layer_norm(x, (8,), w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert y.shape == (0, 8) and gx.shape == (0, 8) and not gw.any() and not gb.any()
    assert F.layer_norm(torch.zeros(3, 0, device="cuda"), (0,)).shape == (3, 0)
    # a constant row is its bias; rows with a NaN or an infinity are NaN and leave the others alone
    x = gen.normal_like(90, 6, 100).cuda()
    clean = ops.layer_norm(x, (100,))[0]
    x[1] = 3.25
    x[2, 17] = float("nan")
    x[4, 99] = float("inf")
    y, mean, rstd = ops.layer_norm(x, (100,))
    assert not y[1].any() and torch.isnan(y[2]).all() and torch.isnan(y[4]).any()
    for r in (0, 3, 5):
        assert torch.equal(y[r], clean[r])
    # eps alone holds the scale of a constant row
    assert float(rstd[1]) == pytest.approx(1e-5 ** -0.5, rel=1e-6)


def test_refusals():
    from repdl_amd import ops
    from repdl_amd.nn import functional as F

    x = torch.zeros(4, 8, device="cuda")
    ok = torch.ones(8, device="cuda")
    bad = [lambda: ops.layer_norm(x.cpu(), (8,)), lambda: ops.layer_norm(x.double(), (8,)), lambda: ops.layer_norm(x, (4,)),
           lambda: ops.layer_norm(x, ()), lambda: ops.layer_norm(x, (4, 8, 1)), lambda: ops.layer_norm(x, (8,), ok[:7]),
           lambda: ops.layer_norm(x, (8,), ok.half()), lambda: ops.layer_norm(x.half(), (8,), ok, ok.half()),
           lambda: ops.layer_norm(x, (8,), ok.cpu()), lambda: ops.layer_norm(x, (8,), ok.view(2, 4)), lambda: F.layer_norm(x, 8, ok.view(1, 8).requires_grad_()), lambda: ops.layer_norm_grad(x, x, ok[:3], ok[:4], (8,)),
           lambda: ops.layer_norm_grad(x.half(), x, ok[:4], ok[:4], (8,)), lambda: ops.layer_norm_grad(x[:3], x, ok[:4], ok[:4], (8,))]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(1, 1), (70, 3), (300, 7), (5, 8), (600, 20), (2000, 63), (37, 64), (1300, 100), (700, 1000), (40, 1025), (9, 2048), (600, 4100),
                                   (5, 8191), (300, 16384), (256, 3), (257, 3), (255, 130), (256, 1000), (257, 1000), (100, 4099), (256, 5000), (64, 16384), (1, 777), (4095, 200),
                                   (4096, 200), (4100, 65), (1100, 5000), (4200, 8200), (50, 64), (50, 65), (300, 72), (300, 73), (50, 96), (50, 97), (300, 144),
                                   (300, 145), (40, 1152), (40, 1153), (300, 1280), (40, 1536), (40, 1537), (300, 2050), (4500, 2056), (20, 9216), (20, 12288), (20, 12289)],
                         ids=str)
def test_bits_of_the_documented_order(shape, kind):
    """Outputs, statistics and all three gradients against a model of the sums' order in numpy's binary32: every bit."""
    from repdl_amd import ops

    t = TYPES[kind]
    x, w, b, gy = data(*shape, t, t, seed=110)
    y, mean, rstd = ops.layer_norm(x, shape[1:], w, b)
    gx, gw, gb = ops.layer_norm_grad(gy, x, mean, rstd, shape[1:], w)
    model = norm_model.LayerNorm(*shape, granule=4 if kind == "f32" else 8)
    args = [v.float().cpu().numpy() for v in (x, w, b, gy)]
    want_y, want_mean, want_rstd, xh = model.forward(args[0], args[1], args[2], 1e-5)
    want_gx, want_gw, want_gb = model.backward(args[3], xh, want_rstd, args[1])
    for got, want in ((mean, want_mean), (rstd, want_rstd), (y, want_y), (gx, want_gx), (gw, want_gw), (gb, want_gb)):
        assert torch.equal(got.cpu(), torch.from_numpy(want).to(got.dtype))


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("cols", [1000, 1280, 2048, 2056, 4096, 8192, 16384])
def test_large_tensors_have_the_bits_of_their_parts(kind, cols):
    """256 MB and more are moved past the caches, by other instructions."""
    from repdl_amd import ops

    t = TYPES[kind]
    rows = (1 << 28) // torch.finfo(t).bits * 8 // cols + 5
    x = gen.normal_like(123, 257, cols).to(t).cuda().repeat(rows // 257 + 1, 1)[:rows]
    w, b = gen.normal_like(124, cols).to(t).cuda(), gen.normal_like(125, cols).to(t).cuda()
    gy = x.flip(0)
    y, mean, rstd = ops.layer_norm(x, (cols,), w, b)
    gx = ops.layer_norm_grad(gy, x, mean, rstd, (cols,), w)[0]
    for at in (slice(0, 300), slice(rows - 300, rows)):
        want = ops.layer_norm(x[at], (cols,), w, b)
        assert torch.equal(y[at], want[0]) and torch.equal(mean[at], want[1]) and torch.equal(rstd[at], want[2])
        assert torch.equal(gx[at], ops.layer_norm_grad(gy[at], x[at], want[1], want[2], (cols,), w)[0])


def test_more_elements_than_32_bits_count():
    from repdl_amd import ops

    rows, cols = (1 << 19) + 3, 4096 + 8           # 2.15e9 elements
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    part = gen.normal_like(120, 64, cols).to(torch.bfloat16).cuda()
    x.copy_(part[:1].expand(rows, cols))
    x[-64:] = part
    w, b = gen.normal_like(121, cols).cuda(), gen.normal_like(122, cols).cuda()
    y, mean, rstd = ops.layer_norm(x, (cols,), w, b)
    want = ops.layer_norm(part, (cols,), w, b)
    assert torch.equal(y[-64:], want[0]) and torch.equal(mean[-64:], want[1]) and torch.equal(y[:1], want[0][:1])
    gx, gw, gb = ops.layer_norm_grad(x, x, mean, rstd, (cols,), w)  # (the rows as their own incoming gradient)
    assert torch.equal(gx[-64:], ops.layer_norm_grad(part, part, want[1], want[2], (cols,), w)[0])
    exact = part.double().sum(0) + part[0].double() * (rows - 64)
    terms = part.double().abs().sum(0) + part[0].double().abs() * (rows - 64)
    # runs of 2050 rows in turn, then 32 + 16 partial sums: at most 2100 roundings, each of at most U of the sum of magnitudes
    assert ((gb.double() - exact).abs() <= 2100 * U * terms).all()


def test_entry_points_with_the_librarys_scratch():
    """The C entry point that brings its own scratch gives the bits of the one that is handed some."""
    import ctypes

    from repdl_amd import _lib, ops

    x, w, b, gy = data(500, 300, torch.float32, torch.float32, seed=130)  # (more than 256 rows: with scratch)
    _, mean, rstd = ops.layer_norm(x, (300,), w, b)
    want = ops.layer_norm_grad(gy, x, mean, rstd, (300,), w)
    got = [torch.empty_like(t) for t in want]
    p = [ctypes.c_void_p(t.data_ptr()) for t in (gy, x, w, mean, rstd, *got)]
    _lib.call("repdl_hip_layer_norm_grad", *p, 500, 300, 0, 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert all(torch.equal(g, v) for g, v in zip(got, want))


def test_side_stream_and_graph():
    from repdl_amd.nn import functional as F

    x, w, b, gy = data(70, 1000, torch.float32, torch.float32, seed=95)
    for t in (x, w, b):
        t.requires_grad_()

    def step():
        y = F.layer_norm(x, (1000,), w, b)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), gy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for rep in range(3):
        with torch.no_grad():
            x.copy_(gen.normal_like(96 + rep, 70, 1000))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(p, q) for p, q in zip(got, step()))


def test_more_threads_than_a_launch_counts():
    """A launch counts its threads in 32 bits: 2^30 rows of four threads, and 2 x 2^27 columns of sixteen, pass that; the rows (columns)
    behind the bound have the bits of those before it."""
    from repdl_amd.nn import functional as F

    rows = gen.normal_like(70, 1 << 18, 2).to(torch.bfloat16).cuda()
    w, b = gen.normal_like(71, 2).cuda(), gen.normal_like(72, 2).cuda()

    def both(x):
        x = x.requires_grad_()
        y = F.layer_norm(x, (2,), w, b)
        return y.detach(), torch.autograd.grad(y, x, x.detach())[0]

    want = both(rows.clone())
    for got, part in zip(both(rows.repeat(4096 + 1, 1)), want):  # (2^30 + 2^18 rows)
        assert (got.view(4096 + 1, -1) == part.view(-1)).all()
    del got
    cols = gen.normal_like(73, 2, 1 << 20).to(torch.bfloat16).cuda()
    x, gy = (c.repeat(129).view(1, -1) for c in cols)
    w, b = (torch.ones(x.shape[1], dtype=torch.bfloat16, device="cuda", requires_grad=True) for _ in range(2))
    gw, gb = torch.autograd.grad(F.layer_norm(x, x.shape[1:], w, b), (w, b), gy)
    assert torch.equal(gb, gy[0]) and gw.any() and (gw.view(129, -1) == gw[:1 << 20]).all()


def test_both_bindings():
    from repdl_amd.backend import hip_ctypes

    try:
        from repdl_amd.backend import _hip_ext
    except ImportError:
        pytest.skip("the compiled binding has not been built")
    x, w, b, gy = data(11, 77, torch.bfloat16, torch.float32, seed=98)
    one, two = (m.layer_norm(x, 77, w, b, 1e-5, True) for m in (hip_ctypes, _hip_ext))
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    assert _hip_ext.layer_norm(x, 77, None, None, 1e-5, False)[1] is None
    one, two = (m.layer_norm_grad(gy, x, one[1], one[2], 77, w, None, True, True, True) for m in (hip_ctypes, _hip_ext))
    assert all(torch.equal(p, q) and p.dtype == q.dtype for p, q in zip(one, two))
