"""Layer normalisation of rows whose level is far above their spread, and of constant rows: forward and gradients against the definition
in binary64 with tolerances that do not grow with the level, the bits of the model, rows of both kinds side by side."""
import numpy as np
import pytest
import torch

import gen
import norm_model_offset

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24
# (level, spread): 1000 to 1000000 times the spread, and around 16 times
LEVELS = [(1000.1, 1.0), (-12345.6, 12.3), (1.0e4, 0.01), (1.0e6, 1.0), (0.7, 0.0001), (15.0, 1.0), (17.0, 1.0), (40.0, 1.0)]
CONSTANTS = [1000.1, 12345.6, 1000000.3, -7.7, 0.3, 1.0e-3, 3.3e7]


def rows_of(rows, cols, kind, seed=1, constants=True):
    """In turn: a row of one of the levels, a constant one, one of no level."""
    x = gen.normal_like(seed, rows, cols)
    for r in range(rows):
        if r % 3 == 0:
            level, spread = LEVELS[r // 3 % len(LEVELS)]
            x[r] = x[r] * spread + level
        elif constants and r % 3 == 1:
            x[r] = CONSTANTS[r // 3 % len(CONSTANTS)]
    t = TYPES[kind]
    if kind == "f16":
        x = x.clamp(-6.0e4, 6.0e4)
    w = (1 + 0.25 * gen.normal_like(seed + 2, cols)).to(t)
    b = (0.5 * gen.normal_like(seed + 3, cols)).to(t)
    return x.to(t), w, b, gen.normal_like(seed + 4, rows, cols).to(t)


def depth(n):
    """Additions on the longest path of a row's sum (at most 24 elements a thread, log2 of the rest), and one more per wave or long stride."""
    return 24 + 6 + 16 + n // 4096


def parts(x, eps):
    """centred x, rstd, normalised x, and the error of the normalised x that a kernel may have, in binary64"""
    x = x.double()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    std = (d * d).mean(1, keepdim=True).sqrt()
    rstd = 1 / torch.sqrt(std * std + eps)
    # A row above 16 times its spread is centred by a mean off by at most a step of the level (u) and then by the mean of
    # what that leaves, at most max|d| + u: depth + 2 roundings of these sizes.  Any other row's one mean is off by as many of its
    # largest value, at most 17 spreads + max|d| (the comparison itself has rounded values: 17, not 16).
    u = 2 * U * mean.abs()
    far = mean.abs() > 17 * std
    size = d.abs().amax(1, keepdim=True) + torch.where(far, u, 17 * std)
    k = depth(x.shape[1])
    xh = d * rstd
    err = (k + 4) * U * size * rstd * (1 + xh.abs()) + xh.abs() * (k + 12) * U
    return d, rstd, xh, err


def check(x, w, b, gy, y, mean, rstd, grads, eps=1e-5):
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal
    constant = (x == x[:, :1]).all(1)
    # a constant row is its bias, to the bit, and its mean is its value
    assert torch.equal(y[constant], b.expand_as(y)[constant]), (y[constant].double() - b.double()).abs().max()
    assert torch.equal(mean[constant], x[constant, 0].float())
    d, r, xh, err = parts(x, eps)
    wd, bd, gyd = w.double(), b.double(), gy.double()
    want = xh * wd + bd
    tol = err * wd.abs() + want.abs() * (2 * U + half) + (xh * wd).abs() * 2 * U + tiny
    off = (y.double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())
    rel = (depth(x.shape[1]) + 12) * U + 2 * (err * xh.abs()).mean(1, keepdim=True)
    assert ((rstd.double()[:, None] - r).abs() <= r * rel).all()
    gx, gw, gb = grads
    g = gyd * wd
    want = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    k = depth(x.shape[1]) + 8
    m = lambda v: v.mean(1, keepdim=True)  # noqa: E731
    tol = r * (k * U * (g.abs() + m(g.abs()) + xh.abs() * m((g * xh).abs())) + err * m((g * xh).abs()) + xh.abs() * m(g.abs() * err))
    tol = tol + want.abs() * (rel + 4 * U + half) + tiny
    off = (gx.double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())
    n = len(x) // 256 + 64 + 48 + 16
    for got, want, size, extra in ((gw, (gyd * xh).sum(0), gyd.abs() * (xh.abs() + err), (gyd.abs() * err).sum(0)), (gb, gyd.sum(0), gyd.abs(), 0.0)):
        tol = n * U * size.sum(0) + extra + want.abs() * half + tiny
        off = (got.double() - want).abs()
        assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("cols", [2, 3, 40, 100, 768, 1001, 5120, 16384])
def test_the_model_keeps_the_bound(cols):
    """The kernels' arithmetic on the CPU: what the bits below are held to is right itself."""
    x, w, b, gy = rows_of(48, cols, "f32")
    model = norm_model_offset.LayerNorm(48, cols, 4)
    args = [v.numpy() for v in (x, w, b, gy)]
    y, mean, rstd, offset = model.forward(args[0], args[1], args[2], 1e-5)
    assert 16 < offset.sum() < 48 or cols < 40
    grads = model.backward(args[3], args[0], mean, rstd, args[1])
    check(x, w, b, gy, *(torch.from_numpy(v) for v in (y, mean, rstd)), [torch.from_numpy(v) for v in grads])


def on_gpu(x, w, b, gy):
    from repdl_amd import ops

    x, w, b, gy = (v.cuda() for v in (x, w, b, gy))
    y, mean, rstd = ops.layer_norm(x, x.shape[1:], w, b)
    return y, mean, rstd, ops.layer_norm_grad(gy, x, mean, rstd, x.shape[1:], w)


SHAPES = [(24, 1), (24, 2), (48, 3), (300, 3), (48, 40), (300, 64), (48, 100), (300, 100), (48, 200), (300, 500), (48, 768), (300, 768), (48, 1001), (300, 1001),
          (25, 1152), (300, 1152), (48, 1500), (301, 1500), (300, 2056), (48, 3000), (300, 3001), (48, 5120), (300, 5120), (25, 12288), (300, 12288), (48, 16384), (257, 16384),
          (24, 16385), (48, 20001), (300, 20000), (24, 70001)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_definition(shape, kind):
    x, w, b, gy = rows_of(*shape, kind)
    y, mean, rstd, grads = on_gpu(x, w, b, gy)
    check(x, w, b, gy, y.cpu(), mean.cpu(), rstd.cpu(), [g.cpu() for g in grads])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1] <= 16384] + [(5000, 100), (4100, 1500)], ids=str)
def test_bits_of_the_model(shape, kind):
    x, w, b, gy = rows_of(*shape, kind, seed=9)
    y, mean, rstd, grads = on_gpu(x, w, b, gy)
    model = norm_model_offset.LayerNorm(*shape, 4 if kind == "f32" else 8)
    args = [v.float().numpy() for v in (x, w, b, gy)]
    want = model.forward(args[0], args[1], args[2], 1e-5)[:3]
    for got, v in zip((y, mean, rstd, *grads), want + model.backward(args[3], args[0], want[1], want[2], args[1])):
        assert torch.equal(got.cpu(), torch.from_numpy(np.ascontiguousarray(v)).to(got.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [3, 40, 100, 500, 1500, 3000, 20000])
def test_rows_do_not_depend_on_their_company(cols):
    """An offset row alone, among its kind and among others; the others keep their bits beside it."""
    from repdl_amd import ops

    x, w, b, gy = (v.cuda() for v in rows_of(270, cols, "f32", seed=20))
    y, mean, rstd = ops.layer_norm(x, (cols,), w, b)
    gx = ops.layer_norm_grad(gy, x, mean, rstd, (cols,), w)[0]
    for at in (slice(0, 1), slice(1, 2), slice(2, 3), slice(3, 9), slice(200, 269), slice(0, 270, 3), slice(2, 270, 3)):
        part = x[at].clone()
        yp, mp, rp = ops.layer_norm(part, (cols,), w, b)
        assert torch.equal(yp, y[at]) and torch.equal(mp, mean[at]) and torch.equal(rp, rstd[at])
        assert torch.equal(ops.layer_norm_grad(gy[at].clone(), part, mp, rp, (cols,), w)[0], gx[at])


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [2, 40, 100, 500, 1500, 3000, 20000])
def test_no_numbers_beside_offset_rows(cols):
    """Rows with an infinity, a NaN, or values whose squares overflow keep their bits beside offset rows."""
    from repdl_amd import ops

    x = gen.normal_like(25, 64, cols)
    x[1::4, 0], x[2::4, cols - 1], x[3::8] = float("inf"), float("nan"), x[3::8] * 1e25
    x = x.cuda()
    bits = lambda t: t.view(torch.int32)  # noqa: E731
    want = ops.layer_norm(x, (cols,))
    gy = gen.normal_like(26, 64, cols).cuda()
    grad = ops.layer_norm_grad(gy, x, want[1], want[2], (cols,))[0]
    x[0::4] = x[0::4] * 1e-3 + 1000.1
    got = ops.layer_norm(x, (cols,))
    others = [r for r in range(64) if r % 4]
    assert all(torch.equal(bits(g[others]), bits(v[others])) for g, v in zip(got, want))
    assert torch.isfinite(got[0][0::4]).all()
    assert torch.equal(bits(ops.layer_norm_grad(gy, x, got[1], got[2], (cols,))[0][others]), bits(grad[others]))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(9, 1001), (300, 1500), (40, 20001)])
def test_only_some_gradients(rows, cols):
    """The sums over rows without gx (a long row's rest is then made for them alone), gx without them: the same bits."""
    from repdl_amd import ops

    x, w, b, gy = (v.cuda() for v in rows_of(rows, cols, "f32", seed=30))
    _, mean, rstd = ops.layer_norm(x, (cols,), w, b)
    want = ops.layer_norm_grad(gy, x, mean, rstd, (cols,), w)
    for which in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        for need, got, v in zip(which, ops.layer_norm_grad(gy, x, mean, rstd, (cols,), w, None, *which), want):
            assert (got is not None) == need and (got is None or torch.equal(got, v))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_tensors_past_the_caches(kind):
    """256 MB and more are read by other instructions: the bits of the parts."""
    from repdl_amd import ops

    cols = 4096
    rows = (1 << 28) // torch.finfo(TYPES[kind]).bits * 8 // cols + 5
    part, w, b, _ = (v.cuda() for v in rows_of(258, cols, kind, seed=40))
    x = part.repeat(rows // 258 + 1, 1)[:rows]
    y, mean, rstd = ops.layer_norm(x, (cols,), w, b)
    gx = ops.layer_norm_grad(x, x, mean, rstd, (cols,), w)[0]
    for at in (slice(0, 300), slice(rows - 300, rows)):
        want = ops.layer_norm(x[at], (cols,), w, b)
        assert torch.equal(y[at], want[0]) and torch.equal(mean[at], want[1]) and torch.equal(rstd[at], want[2])
        assert torch.equal(gx[at], ops.layer_norm_grad(x[at], x[at], want[1], want[2], (cols,), w)[0])


@pytest.mark.gpu
def test_gradients_of_an_offset_row_against_differences():
    """As the definition's slope along a direction (binary64 differences), for rows 1000 times above their spread."""
    from repdl_amd.nn import functional as F

    rows, cols = 12, 77
    x = (gen.normal_like(50, rows, cols) + 1000.1).cuda().requires_grad_()
    w, b = ((gen.normal_like(51 + i, cols) * 0.2 + 1).cuda().requires_grad_() for i in range(2))
    gy = gen.normal_like(53, rows, cols).cuda()
    grads = torch.autograd.grad(F.layer_norm(x, (cols,), w, b), (x, w, b), gy)

    def value(x, w, b):
        d = x - x.mean(1, keepdim=True)
        return (((d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)) * w + b) * gy.double().cpu()).sum()

    args = [t.detach().double().cpu() for t in (x, w, b)]
    for i, g in enumerate(grads):
        v, h = gen.normal_like(60 + i, *g.shape).double(), 1e-5
        up, down = (value(*[a + s * v if j == i else a for j, a in enumerate(args)]) for s in (h, -h))
        want = float((up - down) / (2 * h))
        size = float((g.double().cpu() * v).abs().sum())
        # (the difference: h^2 of the third derivative, and 2^-52 * 1000 / h for the rounded x + h v)
        assert abs(float((g.double().cpu() * v).sum()) - want) <= size * 100 * U + 1e-6
