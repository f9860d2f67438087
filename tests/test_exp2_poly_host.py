"""The polynomials for 2^f of the preference loss: their coefficients are what the table generator makes, near the best that the degree
allows, and a term of a row's sum keeps the bound that follows."""
import os
import re
import subprocess
import sys

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "repdl_amd", "csrc")


def test_coefficients_are_the_generators():
    pytest.importorskip("mpmath")
    sys.path.insert(0, CSRC)
    try:
        import gen_tables
    finally:
        sys.path.remove(CSRC)
    text = open(os.path.join(CSRC, "crmath_tables.h")).read()
    # the best relative error of a polynomial of degree n is near 2 (ln 2 / 4)^(n+1) / (n+1)!: 7.5e-8 and 1.9e-9; exactly 1 at 0 and
    # coefficients of 24 bits (half a step of ln 2 f at f = 1/2: 1.5e-8) cost the rest
    for degree, most in ((5, 1.2e-7), (6, 2.0e-8)):
        coefficients, error = gen_tables.exp2_poly(degree)
        have = [float.fromhex(v[:-1]) for v in re.findall(r"#define CRM_EXP2_%d_C\d (\S+)" % degree, text)]
        assert have == coefficients and float(error) < most


def test_terms_keep_their_bound(tmp_path):
    """|error| of 2^f in binary32 steps: the polynomial's own (1.08e-7 = 1.82 U, 0.27 U), one rounding of up to half a step of a
    result below 1.42 down to 0.7 (1.42 U relative to it), and that of the sum before it, at most 0.42 f -> 0.3 U: below 4 U and 2 U.
    The maximum's own term times the base has the base's 2 U and the rounded m L's ln 2 / 4 U besides."""
    src = tmp_path / "poly.c"
    src.write_text(r'''
#include <stdio.h>
#include "crmath.h"
int main(void)
{
    double worst[4] = {0, 0, 0, 0};
    for (int d = 5; d <= 6; d++)
    {
        for (int i = -5000000; i <= 5000000; i++)
        {
            const float f = (float)(i * 1e-7);
            const double e = fabs((double)crm_exp2_poly(f, d) / exp2((double)f) - 1);
            if (!(e <= worst[d - 5])) worst[d - 5] = e;
        }
        for (int i = -4000000; i <= 4000000; i++)
        {
            const float m = (float)(i * 1e-5), c = crm_exp_shift(m);
            const double e = fabs((double)crm_exp_term(m, c, d) * crm_exp_base(m, c) - 1);
            if (!(e <= worst[d - 3])) worst[d - 3] = e;
        }
    }
    printf("%.4f %.4f %.4f %.4f %d\n", worst[0] * 0x1p24, worst[1] * 0x1p24, worst[2] * 0x1p24, worst[3] * 0x1p24,
           crm_exp2_poly(0.0f, 5) == 1.0f && crm_exp2_poly(0.0f, 6) == 1.0f);
    return 0;
}
''')
    exe = tmp_path / "poly"
    subprocess.run(["gcc", "-O2", "-std=c11", "-ffp-contract=off", "-mfma", "-I", CSRC, str(src), "-o", str(exe), "-lm"], check=True)
    p5, p6, t5, t6, one = (float(v) for v in subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.split())
    assert p5 <= 4 and p6 <= 2 and t5 <= 6.2 and t6 <= 4.2 and one == 1, (p5, p6, t5, t6)
