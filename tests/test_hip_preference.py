"""The preference loss on the GPU: loss, log probabilities and gradient against the definition in binary64 over vocabularies on
both sides of every change of kernel and chunk, in every type; tokens that are not counted; masked vocabularies, infinities and
NaN; strides; refusals; streams, graphs, a run of it with layer norm and dropout."""
import math

import pytest
import torch

import gen

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def reference(logits, target, ref, beta, eps, ignore=-100):
    """loss, logps, gradient, and what the tolerances are made of, in binary64 on the CPU"""
    x = logits.detach().double().cpu()
    t = target.cpu()
    counted = t != ignore
    x = x - x.amax(2, keepdim=True)  # (exact enough in binary64; a large logit minus its logsumexp would lose the logarithm)
    lse = torch.log(torch.exp(x).sum(2))
    lp = x.gather(2, t.clamp(min=0).unsqueeze(2)).squeeze(2) - lse
    logps = torch.where(counted, lp, 0.0).sum(1)
    P = len(x) // 2
    margin = logps - (0 if ref is None else ref.double().cpu())
    z = beta * (margin[:P] - margin[P:])
    loss = (1 - eps) * torch.nn.functional.softplus(-z) + eps * torch.nn.functional.softplus(z)
    c = beta / P * (eps * torch.sigmoid(z) - (1 - eps) * torch.sigmoid(-z))
    coef = torch.cat([c, -c])[:, None, None] * counted[:, :, None]
    p = torch.softmax(x, 2)
    hot = torch.nn.functional.one_hot(t.clamp(min=0), x.shape[2])
    return loss.mean(), logps, coef * (hot - p), (coef, p, hot, counted, z)


def check(loss, logps, grad, logits, target, ref, beta, eps, ignore=-100):
    want, L, g, (coef, p, hot, counted, z) = reference(logits, target, ref, beta, eps, ignore)
    V, P = logits.shape[2], len(L) // 2
    x = logits.detach().double().cpu()
    d = (x - x.amax(2, keepdim=True)).abs()
    # A term exp(x - m) of the sum is off by (8.2 + 0.23 |d|) U (16 bits, a polynomial of degree 5: 4.9e-7 = 8.2 U; 2 + 0.23 |d| in binary32),
    # at most 2.25 |d| U where a large maximum is subtracted first; weighted with the terms the |d| average to at most log V.  The sum
    # adds at most 64 / 4 + 2 + 6 + 3 + V / 16384 roundings, its factor 2^(K - m L) 2.  The rest of a log probability is binary64.
    k = 10.2 + 2.25 * math.log(V) + 27 + V / 16384
    err_L = counted.sum(1) * k * U + 1e-12
    assert ((logps.double().cpu() - L).abs() <= err_L + L.abs() * U).all(), (logps, L)
    err_z = beta * (err_L[:P] + err_L[P:])
    assert abs(float(loss.detach()) - float(want)) <= float(err_z.mean()) + float(want) * 2 * U
    if grad is None:
        return
    # c is off by beta/P err_z / 4 and two roundings; p by its exponential (2 + 2.25 |d|: crm_exp_neg and the rounded difference), the
    # sum, the reciprocal and three products
    err_c = (torch.cat([beta / P * err_z / 4] * 2)[:, None, None] + coef.abs() * 4 * U) * counted[:, :, None]
    tol = err_c * (hot - p).abs() + coef.abs() * p * (2 + 2.25 * d + k + 6) * U + coef.abs() * hot * 2 * U
    # (below the type's normal numbers a step is absolute: half of it; the exponential itself ends at 2^-149)
    tol = tol + g.abs() * (torch.finfo(logits.dtype).eps / 2 + 2 * U) + torch.finfo(logits.dtype).smallest_normal * torch.finfo(logits.dtype).eps + 2.0 ** -126
    assert grad.dtype == logits.dtype and grad.shape == logits.shape and grad.is_contiguous()
    off = (grad.double().cpu() - g).abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert not grad.cpu()[~counted].any()


def data(pairs, steps, vocab, kind, seed=1, holes=True):
    x = (gen.normal_like(seed, 2 * pairs, steps, vocab) * 3).to(TYPES[kind]).cuda()
    t = gen.labels(seed + 1, 2 * pairs * steps, vocab).view(2 * pairs, steps)
    if holes and steps > 2:
        t[0, 0] = t[-1, -1] = t[1, steps // 2] = -100
    ref = -math.log(vocab) * steps + 2 * gen.normal_like(seed + 2, 2 * pairs)
    return x, t.cuda(), ref.cuda()


CASES = [(1, 1, 1), (1, 1, 2), (2, 3, 7), (3, 5, 10), (1, 17, 63), (2, 4, 64), (2, 9, 257), (1, 6, 1000), (2, 5, 1024), (2, 5, 1025), (1, 3, 4095), (2, 3, 4096),
         (1, 3, 4097), (1, 2, 8192), (1, 2, 8193), (2, 2, 16384), (1, 2, 16385), (1, 3, 32000), (1, 2, 50257), (5, 130, 33), (1, 1100, 9), (40, 3, 11)]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_definition(case, kind):
    from repdl_amd.nn import functional as F

    x, t, ref = data(*case, kind)
    x.requires_grad_()
    for r, beta, eps in ((ref, 0.1, 0.0), (None, 0.5, 0.2)):
        loss, logps = F.preference_loss(x, t, r, beta, eps)
        assert loss.shape == () and logps.shape == (2 * case[0],) and not logps.requires_grad
        (g,) = torch.autograd.grad(loss, x)
        check(loss, logps, g, x, t, r, beta, eps)
        with torch.no_grad():  # the form without what the backward pass needs: the same bits
            alone = F.preference_loss(x, t, r, beta, eps)
        assert torch.equal(alone[0], loss.detach()) and torch.equal(alone[1], logps)


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    """preference_model.c as a function of tensors -> loss, logps, row statistics, coefficients"""
    import ctypes
    import os
    import subprocess

    here = os.path.dirname(os.path.abspath(__file__))
    so = str(tmp_path_factory.mktemp("model") / "preference_model.so")
    subprocess.run(["gcc", "-O2", "-std=c11", "-ffp-contract=off", "-mfma", "-shared", "-fPIC", "-I", os.path.join(here, "..", "repdl_amd", "csrc"),
                    os.path.join(here, "preference_model.c"), "-o", so, "-lm"], check=True)
    lib = ctypes.CDLL(so)
    i64, f64 = ctypes.c_int64, ctypes.c_double

    def run(x, t, ref, beta, eps, ignore=-100):
        seqs, steps, vocab = x.shape
        xc, tc = x.detach().float().cpu().contiguous(), t.cpu().contiguous()
        rc = None if ref is None else ref.cpu()
        out = [torch.zeros(()), torch.zeros(seqs), torch.zeros(seqs, steps, 2), torch.zeros(seqs)]
        p = lambda v: None if v is None else ctypes.c_void_p(v.data_ptr())  # noqa: E731
        lib.preference_model(p(xc), p(tc), p(rc), i64(seqs // 2), i64(steps), i64(vocab), 4 if x.dtype == torch.float32 else 8, f64(beta), f64(eps),
                             i64(ignore), *(p(v) for v in out))
        return out

    return run


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("case", CASES + [(1, 700, 70), (3, 2, 40000), (1100, 1, 5), (1, 2, 131072)], ids=str)
def test_bits_of_the_documented_order(case, kind, model):
    from repdl_amd import ops

    x, t, ref = data(*case, kind, seed=33)
    for r, beta, eps in ((ref, 0.1, 0.0), (None, 0.5, 0.2)):
        got = ops.preference_loss(x, t, r, beta, eps)
        for g, want in zip(got, model(x, t, r, beta, eps)):
            g = g.cpu()
            if g.dim() == 3:  # (the statistics of a token that is not counted are not read)
                g, want = g[t.cpu() != -100], want[t.cpu() != -100]
            assert torch.equal(g.view(torch.int32), want.view(torch.int32))
    far = (x.float() * 0.5 - 3.0e6).to(x.dtype) if kind != "f16" else x - 6.0e4  # (beyond the terms' integers: the maximum subtracted first)
    got, want = ops.preference_loss(far, t, ref), model(far, t, ref, 0.1, 0.0)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])


# A launch counts its threads in 32 bits; what lies behind that bound has the bits of what lies before it.
def test_more_pairs_than_a_launch_counts():
    from repdl_amd import ops

    x, t, ref = data(1021, 1, 5, "f32", seed=50)
    small = ops.preference_loss(x, t, ref)
    times = 4109  # (4195289 pairs of 1024 threads)
    wide = [v.view(2, 1021, -1).repeat(1, times, 1).view(2 * 1021 * times, *v.shape[1:]) for v in (x, t, ref)]
    loss, logps, stats, coef = ops.preference_loss(*wide)
    assert (logps.view(2, times, 1021) == small[1].view(2, 1, 1021)).all()
    assert (stats.view(2, times, 1021, 2) == small[2].view(2, 1, 1021, 2)).all()
    # (the sum adds 4097 + 15 + 6 binary64 roundings; the result rounds once, the other's did too: two half steps.  Coefficients alike.)
    assert abs(float(loss) - float(small[0])) <= 2 * (U + 4200 * 2.0 ** -53) * float(small[0])
    assert ((coef.view(2, times, 1021).double() * times - small[3].view(2, 1, 1021).double()).abs() <= 2.001 * U * small[3].view(2, 1, 1021).double().abs()).all()


def test_more_rows_than_a_launch_counts():
    from repdl_amd import ops

    P, steps = 8, 4194310  # (67108960 rows, 64 threads each)
    x = (gen.normal_like(51, 2 * P, 1000, 3) * 3).to(torch.bfloat16).cuda().repeat(1, 4195, 1)[:, :steps]
    t = gen.labels(52, 2 * P * 1000, 3).view(2 * P, 1000).cuda().repeat(1, 4195)[:, :steps].contiguous()
    loss, logps, stats, coef = ops.preference_loss(x, t, None)
    g = torch.ones((), device="cuda")
    gx = ops.preference_loss_grad(x, t, stats, coef, g)
    few = [0, 7, 8, 15]  # the first and the last pair
    alone = ops.preference_loss(x[few], t[few], None)
    assert torch.equal(logps[few], alone[1]) and torch.equal(stats[few], alone[2])
    assert torch.equal(gx[few], ops.preference_loss_grad(x[few], t[few], stats[few], coef[few], g))
    # (over millions of tokens a pair's margin leaves a coefficient of one side or of zero: coefficients of our own show every row)
    coef = torch.linspace(-1.0, 1.0, 2 * P, device="cuda")
    gx = ops.preference_loss_grad(x, t, stats, coef, g)
    assert torch.equal(gx[few], ops.preference_loss_grad(x[few], t[few], stats[few], coef[few], g)) and gx[15, -50:].any()


def test_more_chunks_than_a_launch_counts():
    """One row of logits, seen 16777400 times, 256 threads each."""
    from repdl_amd import ops

    steps, g = 8388700, torch.ones((), device="cuda")
    row = (gen.normal_like(53, 1, 1, 4097) * 3).half().cuda()
    t = torch.full((2, steps), 1001, device="cuda")
    stats = ops.preference_loss(row.expand(2, steps, 4097), t, None)[2]
    assert (stats == ops.preference_loss(row.expand(2, 1, 4097), t[:, :1], None)[2]).all()
    row, coef = row[:, :, :1025], torch.tensor([1.0, -1.0], device="cuda")  # (34 GB of gradients)
    gx = ops.preference_loss_grad(row.expand(2, steps, 1025), t, stats, coef, g)
    want = ops.preference_loss_grad(row.expand(2, 1, 1025), t[:, :1], stats[:, :1], coef, g)
    assert want.any() and (gx[0, :500] == want[0]).all() and (gx[1, :500] == want[1]).all() and (gx[1, -500:] == want[1]).all()


def test_incoming_gradient_scales():
    from repdl_amd.nn import functional as F

    x, t, ref = data(2, 3, 100, "f32")
    x.requires_grad_()
    (g,) = torch.autograd.grad(F.preference_loss(x, t, ref)[0], x)
    (h,) = torch.autograd.grad(F.preference_loss(x, t, ref)[0] * -4.0, x)  # (a power of two: exact)
    assert torch.equal(h, -4.0 * g)


def test_gradient_against_differences():
    """The slope of the binary64 definition along a direction: the difference is off by h^2 of the third derivative and 2^-52 / h
    of the loss, 1e-9 here; the gradient's terms are off by some 50 U."""
    from repdl_amd.nn import functional as F

    x, t, ref = data(3, 5, 60, "f32", seed=20)
    x.requires_grad_()
    (g,) = torch.autograd.grad(F.preference_loss(x, t, ref, 0.3, 0.1)[0], x)
    v = gen.normal_like(25, *x.shape).double()
    h = 1e-5
    up, down = (float(reference(x.detach().double().cpu() + s * v, t, ref, 0.3, 0.1)[0]) for s in (h, -h))
    assert abs(float((g.double().cpu() * v).sum()) - (up - down) / (2 * h)) <= 100 * U * float((g.double().cpu() * v).abs().sum()) + 1e-8


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_strides_of_the_logits(kind):
    from repdl_amd.nn import functional as F

    x, t, ref = data(2, 6, 301, kind, seed=30)

    def both(v):
        v = v.detach().requires_grad_()
        loss, logps = F.preference_loss(v, t, ref)
        return (loss.detach(), logps) + torch.autograd.grad(loss, v)

    want = both(x)
    longer = torch.cat([x, x[:, :1]], 1)[:, :6]                       # without the last step
    padded = torch.cat([x, x[:, :, :12] * 0 + 50], 2)[:, :, :301]      # a padded vocabulary, whose padding is not looked at
    off = torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape)  # one element off every boundary
    swapped = x.transpose(0, 1).contiguous().transpose(0, 1)          # steps outermost
    columns = x.transpose(1, 2).contiguous().transpose(1, 2)          # the vocabulary is not contiguous: copied
    for v in (longer, padded, off, swapped, columns):
        assert all(torch.equal(p, q) for p, q in zip(both(v), want))
    one = x[:1].expand(4, 6, 301)                                     # stride 0 between the sequences
    assert torch.equal(F.preference_loss(one, t[:1].expand(4, 6))[0], F.preference_loss(one.contiguous(), t[:1].expand(4, 6).contiguous())[0])


def test_a_sequence_does_not_depend_on_its_batch():
    from repdl_amd.nn import functional as F

    x, t, ref = data(4, 7, 5000, "f32", seed=40)
    logps = F.preference_loss(x, t, ref)[1]
    for i in range(4):
        two = [i, 4 + i]
        assert torch.equal(F.preference_loss(x[two], t[two], ref[two])[1], logps[two])


def test_tokens_that_are_not_counted_are_not_read():
    from repdl_amd.nn import functional as F

    x, t, ref = data(2, 5, 5000, "f32", seed=50)
    t[1] = -100                      # a whole sequence without tokens
    x.requires_grad_()
    loss, logps = F.preference_loss(x, t, ref)
    (g,) = torch.autograd.grad(loss, x)
    check(loss, logps, g, x, t, ref, 0.1, 0.0)
    assert float(logps[1]) == 0.0
    junk = x.detach().clone()
    junk[t == -100] = float("nan")
    junk.requires_grad_()
    loss2, logps2 = F.preference_loss(junk, t, ref)
    assert torch.equal(loss2, loss) and torch.equal(logps2, logps) and torch.equal(torch.autograd.grad(loss2, junk)[0], g)
    # another ignore_index, also a token's number
    other = torch.where(t == -100, 7, t)
    loss3, logps3 = F.preference_loss(junk, other, ref, ignore_index=7)
    w = torch.where(other == 7, -100, other)
    assert torch.equal(logps3, F.preference_loss(junk, w, ref)[1])
    nothing = torch.full_like(t, -100)
    loss4, logps4 = F.preference_loss(junk, nothing)
    assert not logps4.any() and float(loss4.detach()) == pytest.approx(math.log(2), rel=2 * U)
    assert not torch.autograd.grad(loss4, junk)[0].any()
    loss5, logps5 = F.preference_loss(x[:, :0], t[:, :0])  # no steps at all
    assert not logps5.any() and float(loss5.detach()) == float(loss4.detach())
    (g5,) = torch.autograd.grad(F.preference_loss(x[:, :0], t[:, :0])[0], x)
    assert not g5.any()


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("vocab", [40, 3000, 20000])
def test_masked_vocabulary_and_large_logits(vocab, kind):
    """-inf or the type's lowest value in masked places: no probability, a gradient of exactly 0; logits far from 0."""
    from repdl_amd.nn import functional as F

    x, t, ref = data(2, 3, vocab, kind, seed=60)
    for fill in (-float("inf"), torch.finfo(TYPES[kind]).min):
        y = x.clone()
        masked = torch.zeros(vocab, dtype=torch.bool, device="cuda")
        masked[::3] = True
        y[:, :, masked] = fill
        tt = torch.where((t >= 0) & (t % 3 == 0), torch.where(t + 1 < vocab, t + 1, 1), t)
        y[0, 1] = fill
        y[0, 1, tt[0, 1]] = 1.0        # one possible token
        y = y.requires_grad_()
        loss, logps = F.preference_loss(y, tt, ref)
        (g,) = torch.autograd.grad(loss, y)
        assert torch.isfinite(logps).all() and torch.isfinite(loss)
        assert not g[:, :, masked].any() and torch.isfinite(g).all()
        z = torch.where(torch.isinf(y.detach()), torch.finfo(TYPES[kind]).min, y.detach().float()).to(y.dtype)
        check(loss, logps, g, z, tt, ref, 0.1, 0.0)
    big = (x.float() * 0 + 1000.0 + 3 * gen.normal_like(65, *x.shape).cuda()).to(TYPES[kind]).requires_grad_()
    loss, logps = F.preference_loss(big, t, ref)
    check(loss, logps, torch.autograd.grad(loss, big)[0], big, t, ref, 0.1, 0.0)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("vocab", [40, 3000, 20000])
def test_rows_of_one_value(vocab, kind):
    """Every logit the same -- the type's lowest value, its largest, 0 --: each token has probability 1 / V."""
    from repdl_amd.nn import functional as F

    t = gen.labels(66, 4, vocab).view(2, 2).cuda()
    for value in (torch.finfo(TYPES[kind]).min, torch.finfo(TYPES[kind]).max, 0.0, -3.0e4, 2.0 ** 21 if kind != "f16" else 2.0 ** 15):
        y = torch.full((2, 2, vocab), value, dtype=TYPES[kind], device="cuda", requires_grad=True)
        loss, logps = F.preference_loss(y, t)
        check(loss, logps, torch.autograd.grad(loss, y)[0], y, t, None, 0.1, 0.0)


@pytest.mark.parametrize("vocab", [50, 3000, 20000])
def test_what_is_not_a_number(vocab):
    """A NaN, a +inf, a row of nothing but -inf, a target outside the vocabulary: NaN for that sequence, the loss and its pair's
    gradient; the other pairs keep theirs."""
    from repdl_amd.nn import functional as F

    x, t, ref = data(3, 4, vocab, "f32", seed=70, holes=False)
    clean = F.preference_loss(x, t, ref)[1]
    for what in ("nan", "inf", "none", "target", "negative"):
        y, tt = x.clone(), t.clone()
        if what == "nan":
            y[1, 2, vocab - 1] = float("nan")
        elif what == "inf":
            y[1, 2, (int(t[1, 2]) + 1) % vocab] = float("inf")
        elif what == "none":
            y[1, 2] = -float("inf")
        else:
            tt[1, 2] = vocab if what == "target" else -7
        y.requires_grad_()
        loss, logps = F.preference_loss(y, tt, ref)
        (g,) = torch.autograd.grad(loss, y)
        keep = [0, 2, 3, 4, 5]
        assert torch.isnan(loss) and torch.isnan(logps[1]) and torch.equal(logps[keep], clean[keep]), what
        assert torch.isnan(g[1]).any() and torch.isnan(g[4]).any() and torch.isfinite(g[[0, 2, 3, 5]]).all(), what
    y = x.clone()
    y[1, 2, t[1, 2]] = -float("inf")     # a token that cannot be: its sequence has probability 0, the loss is infinite
    loss, logps = F.preference_loss(y, t, ref)
    assert float(logps[1]) == -float("inf") and float(loss) == float("inf")


def test_extreme_margins():
    """z from -1e4 to 1e4: softplus without overflow, and with its relative accuracy where it is small."""
    from repdl_amd.nn import functional as F

    x, t, _ = data(1, 2, 10, "f32", seed=80)
    x.requires_grad_()
    for m in (-1e4, -700.0, -90.0, -20.0, -1.0, 0.0, 1.0, 14.0, 20.0, 50.0, 90.0, 1e4):
        ref = torch.tensor([-m, 0.0], device="cuda")
        for eps in (0.0, 0.1):
            loss, logps = F.preference_loss(x, t, ref, 1.0, eps)
            want, _, g, (coef, _, _, _, z) = reference(x, t, ref, 1.0, eps)
            err_z = 4 * (10.2 + 2.25 * math.log(10) + 27) * U  # (as in check(); exp(-z) has z's error as its relative one)
            assert abs(float(loss.detach()) - float(want)) <= float(want) * (err_z + 2 * U) + 2.0 ** -149
            got = torch.autograd.grad(loss, x)[0].double().cpu()
            rel = err_z + 100 * U
            assert ((got - g).abs() <= g.abs() * rel + coef.abs() * 60 * U + 2.0 ** -126).all()


def test_many_pairs_in_order():
    """More pairs than threads in a workgroup: the mean over the pairs is theirs, the same at every call."""
    from repdl_amd import ops

    x, t, ref = data(1500, 1, 3, "f32", seed=85, holes=False)
    loss, logps, _, _ = ops.preference_loss(x, t, ref)
    check(loss, logps, None, x, t, ref, 0.1, 0.0)
    for _ in range(5):
        again = ops.preference_loss(x, t, ref)
        assert torch.equal(again[0], loss) and torch.equal(again[1], logps)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("vocab", [6000, 20480])
def test_large_tensors_have_the_bits_of_their_parts(vocab, kind):
    """256 MB and more are moved past the caches, by other instructions: two pairs against each alone, whose gradient is twice as large."""
    from repdl_amd import ops

    t = TYPES[kind]
    S = (1 << 28) // torch.finfo(t).bits * 8 // (4 * vocab) + 1
    x = gen.normal_like(90, 4, 64, vocab).mul(2).to(t).cuda().repeat(1, S // 64 + 1, 1)[:, :S].contiguous()
    target = gen.labels(91, 4 * S, vocab).view(4, S).cuda()
    target[:, S // 2:S // 2 + 9] = -100
    one = torch.ones((), device="cuda")
    loss, logps, stats, coef = ops.preference_loss(x, target, None, 1e-3)
    g = ops.preference_loss_grad(x, target, stats, coef, one)
    for pair in ([0, 2], [1, 3]):
        px, pt = x[pair], target[pair]
        _, plogps, pstats, pcoef = ops.preference_loss(px, pt, None, 1e-3)
        assert torch.equal(plogps, logps[pair]) and torch.equal(pcoef, 2 * coef[pair])
        assert torch.equal(ops.preference_loss_grad(px, pt, pstats, pcoef, one * 0.5), g[pair])


@pytest.mark.parametrize("V", [65536, 65536 + 3])
def test_more_elements_than_32_bits_count(V):
    from repdl_amd import ops

    P, S = 2, 8200                                    # 2.15e9 elements
    x = torch.zeros(2 * P, S, V, dtype=torch.bfloat16, device="cuda")
    tail = gen.normal_like(86, 8, V).to(torch.bfloat16).cuda()
    x[-1, -8:] = tail
    t = torch.full((2 * P, S), -100, device="cuda")
    t[-1, -8:] = gen.labels(87, 8, V).cuda()
    loss, logps, stats, coef = ops.preference_loss(x, t)
    g = ops.preference_loss_grad(x, t, stats, coef, torch.ones((), device="cuda"))
    small, ts = x[:, -8:].clone(), t[:, -8:].clone()  # the same tokens alone
    loss2, logps2, stats2, coef2 = ops.preference_loss(small, ts)
    assert torch.equal(loss, loss2) and torch.equal(logps, logps2)
    assert torch.equal(g[:, -8:], ops.preference_loss_grad(small, ts, stats2, coef2, torch.ones((), device="cuda")))
    assert not g[:, :-8].any()


def test_entry_point_with_the_librarys_scratch():
    """The C entry point that brings its own scratch gives the bits of the one that is handed some."""
    import ctypes

    from repdl_amd import _lib, ops

    x, t, ref = data(2, 5, 9000, "f32", seed=88)
    want = ops.preference_loss(x, t, ref, 0.1, 0.1)
    got = [torch.zeros_like(v) for v in want]
    p = lambda v: ctypes.c_void_p(v.data_ptr())  # noqa: E731
    _lib.call("repdl_hip_preference_loss", p(x), p(t), p(ref), *(p(v) for v in got), 2, 5, 9000, 5 * 9000, 9000, 0.1, 0.1, -100, 0,
              ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[3], want[3])
    assert torch.equal(got[2][t != -100], want[2][t != -100])


def test_side_stream_and_graph():
    from repdl_amd.nn import functional as F

    x, t, ref = data(3, 6, 2000, "bf16", seed=90)
    x.requires_grad_()

    def step():
        loss, logps = F.preference_loss(x, t, ref)
        return (loss.detach(), logps) + torch.autograd.grad(loss, x)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, step()))
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        graphs.append((graph, held))
    for rep in range(3):
        with torch.no_grad():
            x.copy_(gen.normal_like(91 + rep, *x.shape))
        for graph, held in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, held in graphs:
            assert all(torch.equal(p, q) for p, q in zip(held, want))


def test_refusals():
    from repdl_amd import ops
    from repdl_amd.nn import functional as F

    x, t, ref = data(2, 3, 10, "f32")
    bad = [lambda: ops.preference_loss(x.cpu(), t), lambda: ops.preference_loss(x.double(), t), lambda: ops.preference_loss(x[:3], t[:3]),
           lambda: ops.preference_loss(x[:0], t[:0]), lambda: ops.preference_loss(x[0], t[0]), lambda: ops.preference_loss(x[:, :, :0], t),
           lambda: ops.preference_loss(x, t.int()), lambda: ops.preference_loss(x, t[:, :2]), lambda: ops.preference_loss(x, t.cpu()),
           lambda: ops.preference_loss(x, t, ref[:3]), lambda: ops.preference_loss(x, t, ref.double()), lambda: ops.preference_loss(x, t, ref.cpu()),
           lambda: ops.preference_loss(x, t, ref, -1.0), lambda: ops.preference_loss(x, t, ref, 0.1, 1.0),
           lambda: ops.preference_loss(x, t, ref, 0.1, float("nan")), lambda: ops.preference_loss(x, t, ref, float("nan"))]
    for call in bad:
        with pytest.raises((RuntimeError, ValueError)):
            call()
    with pytest.raises(NotImplementedError):
        F.preference_loss(x, t, ref.requires_grad_())
    loss, logps, stats, coef = ops.preference_loss(x, t)
    for args in ((x, t, stats[:2], coef, loss), (x, t, stats, coef[:2], loss), (x, t, stats, coef, logps)):
        with pytest.raises(RuntimeError):
            ops.preference_loss_grad(*args)


def test_both_bindings():
    from repdl_amd.backend import hip_ctypes

    try:
        from repdl_amd.backend import _hip_ext
    except ImportError:
        pytest.skip("the compiled binding has not been built")
    x, t, ref = data(2, 3, 1234, "f16")
    one, two = (m.preference_loss(x, t, ref, 0.1, 0.1, -100, True) for m in (hip_ctypes, _hip_ext))
    assert all(torch.equal(p[t != -100] if p.dim() == 3 else p, q[t != -100] if q.dim() == 3 else q) for p, q in zip(one, two))
    g = torch.tensor(2.0, device="cuda")
    assert torch.equal(hip_ctypes.preference_loss_grad(x, t, one[2], one[3], g, -100), _hip_ext.preference_loss_grad(x, t, two[2], two[3], g, -100))
    assert _hip_ext.preference_loss(x, t, None, 0.1, 0.1, -100, False)[2] is None


def test_training_a_small_model():
    """Embedding -> (layer norm -> linear -> relu -> linear -> dropout + residual) x 2 -> layer norm -> linear, trained on the
    preference loss: eager steps, and the same steps as one graph's replays, give the same weights; a second run the same again."""
    import repdl_amd
    from repdl_amd import nn, optim
    from repdl_amd.nn import functional as F

    V, D, P, S = 211, 48, 3, 12

    class Block(torch.nn.Module):
        def __init__(self, seed):
            super().__init__()
            self.norm, self.up, self.down, self.drop = nn.LayerNorm(D), nn.Linear(D, 2 * D), nn.Linear(2 * D, D), nn.Dropout(0.1, seed=seed)

        def forward(self, h):
            return self.drop(self.down(torch.relu(self.up(self.norm(h)))), h)

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.table = torch.nn.Parameter(gen.normal_like(1, V, D))
            self.blocks = torch.nn.ModuleList([Block(10), Block(11)])
            self.norm, self.head = nn.LayerNorm(D), nn.Linear(D, V)

        def forward(self, hot):
            h = F.linear(hot, self.table.t().contiguous())  # one-hot rows: a product instead of a gather, whose gradient has no atomics
            for b in self.blocks:
                h = b(h)
            return self.head(self.norm(h)).view(2 * P, S, V)

    tokens = gen.labels(3, 2 * P * S, V).view(2 * P, S).cuda()
    target = torch.cat([tokens[:, 1:], torch.full((2 * P, 1), -100, device="cuda")], 1)
    hot = torch.nn.functional.one_hot(tokens.view(-1), V).float()
    lossf = nn.PreferenceLoss(beta=0.2)
    repdl_amd.init()

    def make():
        torch.manual_seed(5)
        m = Model().cuda()
        return m, optim.SGD(m.parameters(), 0.05)

    def steps(m, opt, n):
        for _ in range(n):
            opt.zero_grad(set_to_none=True)
            lossf(m(hot), target)[0].backward()
            opt.step()

    m, opt = make()
    steps(m, opt, 6)
    want = repdl_amd.utils.get_hash(m)
    assert all(torch.isfinite(p).all() and p.grad is not None and p.grad.abs().sum() > 0 for p in m.parameters())
    m, opt = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        steps(m, opt, 2)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    opt.zero_grad(set_to_none=True)
    with torch.cuda.graph(graph):
        lossf(m(hot), target)[0].backward()
        opt.step()
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert repdl_amd.utils.get_hash(m) == want
