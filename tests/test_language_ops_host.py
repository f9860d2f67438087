"""Layer norm, dropout and the preference loss where no GPU is needed: the C entry points refuse what they cannot take before
anything is launched, the size queries are host arithmetic, the Python layer refuses CPU tensors, and the binary32
exponential of the loss (crm_exp_neg) keeps its bound when compiled for the CPU."""
import ctypes
import os
import subprocess

import pytest
import torch

import philox
import repdl_amd
from repdl_amd import _lib, ops
from repdl_amd.nn import functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p
A = P(0x7F0000000000)  # never dereferenced: every call below ends on the host


def test_layer_norm_arguments():
    lib = _lib.lib()
    assert lib.repdl_hip_layer_norm(None, None, None, None, None, None, 4, 8, 1e-5, 0, 0, None) == -1
    assert lib.repdl_hip_layer_norm(A, None, None, A, A, None, 4, 8, 1e-5, 0, 0, None) == -1   # mean without rstd
    assert lib.repdl_hip_layer_norm(A, None, None, A, None, None, -4, 8, 1e-5, 0, 0, None) == -1
    assert lib.repdl_hip_layer_norm(A, None, None, A, None, None, 4, 8, 1e-5, 3, 0, None) == -1   # no such type
    assert lib.repdl_hip_layer_norm(A, None, None, A, None, None, 4, 8, 1e-5, 0, 1, None) == -1   # binary32 rows, 16-bit weight
    assert lib.repdl_hip_layer_norm(A, None, None, A, None, None, 4, 8, 1e-5, 1, 2, None) == -1
    assert lib.repdl_hip_layer_norm(A, None, None, A, None, None, 4, 1 << 40, 1e-5, 0, 0, None) == -1
    assert lib.repdl_hip_layer_norm(None, None, None, None, None, None, 0, 8, 1e-5, 0, 0, None) == 0
    assert lib.repdl_hip_layer_norm(None, None, None, None, None, None, 4, 0, 1e-5, 0, 0, None) == 0
    assert lib.repdl_hip_layer_norm_grad(None, A, A, A, A, A, A, A, 4, 8, 0, 0, None) == -1
    assert lib.repdl_hip_layer_norm_grad_ws(A, A, A, A, A, A, A, A, 400, 8, 0, 0, None, 0, None) == -3
    assert lib.repdl_hip_layer_norm_grad_ws(A, A, A, A, A, A, A, A, 400, 8, 0, 0, A, 16, None) == -3
    assert lib.repdl_hip_layer_norm_grad_ws(A, A, A, A, A, None, None, None, 4, 8, 0, 0, None, 0, None) == 0  # nothing is wanted
    need = lib.repdl_hip_layer_norm_grad_workspace_bytes
    assert need(0, 8) == 0 and need(8, 0) == 0 and need(-1, 8) == 0
    assert need(1, 1) == 0 and need(256, 16384) == 0  # few rows: one launch, no partial sums
    for rows, cols in ((1, 20000), (257, 1000), (8192, 1024), (100000, 20000)):
        assert 8 * cols <= need(rows, cols) <= 512 * 8 * cols + 512 and need(rows, cols) == need(rows, cols)


def test_dropout_arguments():
    lib = _lib.lib()
    assert lib.repdl_hip_dropout(None, None, A, 8, 0.5, None, 1, 2, 0, None) == -1
    assert lib.repdl_hip_dropout(A, None, None, 8, 0.5, None, 1, 2, 0, None) == -1
    assert lib.repdl_hip_dropout(A, None, A, -8, 0.5, None, 1, 2, 0, None) == -1
    assert lib.repdl_hip_dropout(A, None, A, 1 << 62, 0.5, None, 1, 2, 0, None) == -1
    for p in (-0.1, 1.0001, float("nan"), float("inf")):
        assert lib.repdl_hip_dropout(A, None, A, 8, p, None, 1, 2, 0, None) == -1
    assert lib.repdl_hip_dropout(A, None, A, 8, 0.5, None, 1, 2, 7, None) == -1
    assert lib.repdl_hip_dropout(None, None, None, 0, 0.5, None, 1, 2, 0, None) == 0
    assert lib.repdl_hip_dropout_next_call(None, A, None) == -1
    with pytest.raises(ValueError):
        F.dropout(torch.zeros(3), 1.5, (1, 2))
    for state in (True, None, 3, (1, 2, 3)):  # (what torch's third argument would be, among others)
        with pytest.raises(TypeError):
            ops._dropout_state(state)
    x = torch.zeros(3)
    assert F.dropout(x, 0.5, (1, 2), training=False) is x


def test_preference_arguments():
    lib = _lib.lib()

    def call(pairs=2, steps=3, vocab=10, seq=30, step=10, dtype=0, logits=A, target=A, loss=A, logps=A):
        return lib.repdl_hip_preference_loss_ws(logits, target, None, loss, logps, None, None, pairs, steps, vocab, seq, step, 0.1, 0.0, -100,
                                                dtype, None, 0, None)

    assert call() == -3                      # the workspace is missing: everything else is in order
    for kw in (dict(pairs=0), dict(steps=-1), dict(vocab=0), dict(seq=-1), dict(step=-1), dict(dtype=3), dict(logits=None), dict(target=None),
               dict(loss=None), dict(logps=None), dict(pairs=1 << 31), dict(steps=1 << 31), dict(pairs=1 << 20, steps=1 << 12)):
        assert call(**kw) == -1, kw
    need = lib.repdl_hip_preference_loss_workspace_bytes
    assert need(0, 3, 10) == 0 and need(2, 3, 0) == 0
    assert 2 * 2 * 3 * 12 + 16 <= need(2, 3, 10) <= 2 * 2 * 3 * 12 + 16 + 512
    assert 16 * 512 * (8 * 8 + 4) <= need(8, 512, 131072) <= 16 * 512 * (8 * 8 + 4) + 1024
    assert lib.repdl_hip_preference_loss_grad(A, A, A, A, None, A, 2, 3, 10, 30, 10, -100, 0, None) == -1
    assert lib.repdl_hip_preference_loss_grad(None, None, None, None, None, None, 2, 0, 10, 30, 10, -100, 0, None) == 0


def test_cpu_tensors_are_refused():
    x, t = torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: ops.layer_norm(x, (4,)), lambda: F.layer_norm(x, 4), lambda: ops.dropout(x, 0.5, (1, 2)),
                 lambda: repdl_amd.nn.Dropout(0.5)(x), lambda: repdl_amd.nn.LayerNorm(4)(x), lambda: ops.preference_loss(x, t),
                 lambda: repdl_amd.nn.PreferenceLoss()(x, t), lambda: ops.dropout_next_call(t[0, :2])):
        with pytest.raises(RuntimeError):
            call()


def test_modules_without_a_device():
    """What the layers hold, and what the conversion makes of torch's: only on request."""
    d = repdl_amd.nn.Dropout(0.3, seed=9)
    assert d.rng_state.tolist() == [9, 0] and not d.state_dict()
    x = torch.ones(4)
    assert d.eval()(x) is x and torch.equal(d(x, x), 2 * x)
    with pytest.raises(ValueError):
        repdl_amd.nn.Dropout(0.3, seed=-1)
    net = torch.nn.Sequential(torch.nn.LayerNorm(6, eps=1e-3, bias=False), torch.nn.Dropout(0.2), torch.nn.LayerNorm(6, elementwise_affine=False))
    same = repdl_amd.from_torch_module(net)
    assert [type(m) for m in same] == [type(m) for m in net]
    new = repdl_amd.from_torch_module(net.eval(), language_layers=True)
    assert [type(m).__module__.split(".")[0] for m in new] == ["repdl_amd"] * 3
    assert new[0].bias is None and new[0].eps == 1e-3 and new[2].weight is None and new[1].p == 0.2 and not new[1].training
    assert torch.equal(new[0].weight, net[0].weight) and new[0].weight is not net[0].weight


def test_generator_known_answers():
    """The vectors published with the generator."""
    assert [int(v) for v in philox.block([0] * 4, (0, 0))] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert [int(v) for v in philox.block([0xFFFFFFFF] * 4, (0xFFFFFFFF,) * 2)] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_exponential_keeps_its_bound(tmp_path):
    """crm_exp_neg over every 61st binary32 number in [-110, 0] and the ends: |error| <= (2^-23 + 1.25 |d| 2^-24) exp(d) + half of the
    smallest subnormal step; +0 for -inf, NaN and everything below -105.  The terms: the polynomial's 8.2e-8 < 2^-23; the product
    d * log2(e) rounded to half a step, |d log2(e)| 2^-24, times ln 2; and log2(e) as binary32 has it, 1.44269502163 for 1.44269504089,
    1.335e-8 = 0.224 * 2^-24 too small, which is a factor exp(-1.335e-8 |d|)."""
    src = tmp_path / "exp_neg.c"
    src.write_text(r'''
#include <stdio.h>
#include "crmath.h"
int main(void)
{
    double worst = 0;
    long bad = 0, n = 0;
    const float low = -110.0f;
    for (uint32_t u = 0x80000000u; u <= crm_f2u(low); u += 61)
    {
        const float d = crm_u2f(u);
        const double want = exp((double)d), got = crm_exp_neg(d);
        const double tol = want * (0x1p-23 + fabs((double)d) * 1.25 * 0x1p-24) + 0x1p-150;
        const double off = fabs(got - want) / tol;
        n++;
        if (off > worst) worst = off;
        if (!(off <= 1.0)) bad++;
        if (d < -105.0f && got != 0) bad++;
    }
    if (crm_exp_neg(0.0f) != 1.0f || crm_exp_neg(-0.0f) != 1.0f || crm_exp_neg(-INFINITY) != 0.0f || crm_exp_neg(NAN) != 0.0f
        || crm_exp_neg(-3.0e38f) != 0.0f) bad++;
    printf("%ld %ld %.3f\n", n, bad, worst);
    return 0;
}
''')
    exe = tmp_path / "exp_neg"
    subprocess.run(["gcc", "-O2", "-std=c11", "-ffp-contract=off", "-mfma", "-I", os.path.join(ROOT, "repdl_amd", "csrc"), str(src), "-o", str(exe), "-lm"], check=True)
    n, bad, worst = subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.split()
    assert int(n) > 10 ** 7 and int(bad) == 0, (n, bad, worst)


def test_terms_of_the_row_sum_keep_their_bound(tmp_path):
    """crm_exp_term with crm_exp_base, for maxima of every size up to 2^21 of either sign and x from m down to m - 86.  The product is
    exp(x - m) to 2^-23 (degree 6; 2^-21 for degree 5), 0.224 |x - m| 2^-24 for binary32's log2(e), below 2^-24 for the rounding of
    f (|f| <= 1/2 to 2^-26, times ln 2), and for the base 2^-25 ln 2 of the rounded m L - K and its polynomial's 2^-23: four 2^-24 in all
    beside the first two terms."""
    src = tmp_path / "exp_term.c"
    src.write_text(r'''
#include <stdio.h>
#include "crmath.h"
int main(void)
{
    double worst[2] = {0, 0};
    long bad = 0, n = 0;
    uint32_t r = 12345u;
    for (int i = 0; i < 400000; i++)
    {
        r = r * 1664525u + 1013904223u;
        const float size = ldexpf(1.0f + (float)(r >> 9) * 0x1p-23f, (int)((r >> 3) % 42u) - 21);
        const float m = (r & 1) ? size : -size;
        const float c = crm_exp_shift(m);
        const double base = crm_exp_base(m, c);
        for (int j = 0; j < 24; j++)
        {
            r = r * 1664525u + 1013904223u;
            float x = j == 0 ? m : (j == 1 ? m - 86.0f : m - 86.0f * (float)(r >> 8) * 0x1p-24f);
            if (x < m - 86.0f) x = m - 86.0f;
            const double want = exp((double)x - (double)m);
            for (int d = 5; d <= 6; d++)
            {
                const double got = (double)crm_exp_term(x, c, d) * base;
                const double tol = want * ((d == 6 ? 0x1p-23 : 0x1p-21) + (0.25 * ((double)m - (double)x) + 4.0) * 0x1p-24);
                const double off = fabs(got - want) / tol;
                n++;
                if (off > worst[d - 5]) worst[d - 5] = off;
                if (!(off <= 1.0)) bad++;
            }
        }
    }
    printf("%ld %ld %.3f %.3f\n", n, bad, worst[0], worst[1]);
    return 0;
}
''')
    exe = tmp_path / "exp_term"
    subprocess.run(["gcc", "-O2", "-std=c11", "-ffp-contract=off", "-mfma", "-I", os.path.join(ROOT, "repdl_amd", "csrc"), str(src), "-o", str(exe), "-lm"], check=True)
    n, bad, w5, w6 = subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.split()
    assert int(n) > 10 ** 7 and int(bad) == 0, (n, bad, w5, w6)
