"""Generates ``crmath_tables.h``: the lookup tables of the exp and log kernels.

Run ``python repdl_amd/csrc/gen_tables.py`` after changing a table parameter;
the generated header is committed so that building needs no mpmath.

exp table (128 entries, two 64-bit words each), the published layout of the
binary64 exp of glibc >= 2.28 (sysdeps/ieee754/dbl-64/e_exp_data.c, N = 128):
    2^(k/N) ~= H[k] * (1 + T[k]),  H[k] = RN64(2^(k/N)),  T[k] = RN64(2^(k/N)/H[k] - 1)
    tab[2k]   = bits(T[k])
    tab[2k+1] = bits(H[k]) - (k << 52) / N
so that bits(H[k] * 2^(ki div N)) = tab[2k+1] + (ki << (52 - 7)) for ki = N*m + k.

log tables (128 entries, three separate arrays so that a random entry costs few LDS
bank conflicts: invc as binary32, logc_hi as binary64, logc_lo as binary32).  The argument is reduced to
z in [0.6875, 1.375) and split by the top 7 bits below the leading one of
(bits(z) - bits(0.6875)) into 128 intervals (80 of width 2^-8 below 1, 48 of
width 2^-7 above).  For interval i with centre c:
    invc     = 1/c rounded to 24 significant bits (so z*invc - 1 is exact for a
               24-bit z), exactly 1 for the two intervals that touch 1.0;
    logc_hi  = -log(invc) rounded to a multiple of 2^-43 (k*LN2_HI + logc_hi is
               then exact in binary64);
    logc_lo  = RN32(-log(invc) - logc_hi)  (below 2^-44, so binary32 keeps it to 2^-68).

polynomials for 2^f in binary32, |f| <= 1/2, of degree 5 and 6 (crm_exp_neg, crm_exp_term): minimax in the relative error
among those that are exactly 1 at f = 0, coefficients rounded to binary32.
"""
from __future__ import annotations

import os
import struct

import mpmath as mp

mp.mp.prec = 300
HERE = os.path.dirname(os.path.abspath(__file__))


def bits(x: float) -> int:
    return struct.unpack("<Q", struct.pack("<d", x))[0]


def from_bits(u: int) -> float:
    return struct.unpack("<d", struct.pack("<Q", u))[0]


def rn(x) -> float:
    return float(mp.mpf(x))  # mpmath -> float conversion rounds to nearest even


def round_to_bits(x, nbits: int):
    """Round an mpf to nbits significant bits (nearest)."""
    m, e = mp.frexp(x)
    return mp.ldexp(mp.nint(mp.ldexp(m, nbits)), int(e) - nbits)


def exp_table() -> list[int]:
    N = 128
    tab = []
    for k in range(N):
        v = mp.mpf(2) ** (mp.mpf(k) / N)
        H = rn(v)
        T = rn(v / mp.mpf(H) - 1)
        tab.append(bits(T))
        tab.append(bits(H) - ((k << 52) // N))
    return tab


def log_table():
    OFF = 0x3FE6000000000000
    rows = []
    for i in range(128):
        lo = from_bits(OFF + (i << 45))
        hi = from_bits(OFF + ((i + 1) << 45))
        if i in (79, 80):
            invc = mp.mpf(1)
        else:
            c = (mp.mpf(lo) + mp.mpf(hi)) / 2
            invc = round_to_bits(1 / c, 24)
        logc = -mp.log(invc)
        logc_hi = mp.nint(mp.ldexp(logc, 43)) / mp.mpf(2) ** 43
        logc_lo = logc - logc_hi
        lo32 = struct.unpack("<f", struct.pack("<f", rn(logc_lo)))[0]  # binary64 -> binary32 (innocuous double rounding)
        rows.append((rn(invc), rn(logc_hi), lo32))
        assert mp.mpf(rows[-1][0]) == invc and mp.mpf(rows[-1][1]) == logc_hi
        assert struct.unpack("<f", struct.pack("<f", rows[-1][0]))[0] == rows[-1][0]  # invc is a binary32 number
    return rows


def exp2_poly(degree: int):
    """Coefficients c_1 .. c_degree of the polynomial 1 + c_1 f + ... whose largest relative error against 2^f, |f| <= 1/2, is least,
    rounded to binary32, and the error then.  Remez's exchange: e(f) = 2^-f (1 + c_1 f + ...) - 1 is f times a weighted polynomial, so
    at the best coefficients e(f) / f takes the bound of e with alternating signs at degree + 1 points; each step solves for
    coefficients and bound at the points it has, then moves them to where |e| is largest in each run of one sign of e(f) / f."""
    grid = [mp.mpf(i) / 4000 for i in range(-2000, 2001) if i != 0]
    points = [mp.cos(mp.pi * (2 * i + 1) / (2 * degree + 2)) / 2 for i in reversed(range(degree + 1))]
    points = [f if abs(f) > 0.01 else mp.mpf("0.05") for f in points]

    def error(c, f):
        return mp.mpf(2) ** -f * mp.polyval(c[::-1] + [1], f) - 1

    for _ in range(30):
        rows, right = mp.matrix(degree + 1, degree + 1), mp.matrix(degree + 1, 1)
        for i, f in enumerate(points):
            for j in range(degree):
                rows[i, j] = mp.mpf(2) ** -f * f ** (j + 1)
            rows[i, degree] = (-1) ** i * (-1 if f < 0 else 1)
            right[i] = 1 - mp.mpf(2) ** -f
        solution = list(mp.lu_solve(rows, right))
        runs = []
        for f in grid:
            e = error(solution[:degree], f)
            if not runs or (runs[-1][1] * runs[-1][0] > 0) != (e * f > 0):
                runs.append((f, e))
            elif abs(e) > abs(runs[-1][1]):
                runs[-1] = (f, e)
        assert len(runs) == degree + 1
        points = [f for f, _ in runs]
        if max(abs(e) for _, e in runs) <= abs(solution[degree]) * (1 + mp.mpf(10) ** -4):
            break
    rounded = [round_to_bits(c, 24) for c in solution[:degree]]
    return [rn(c) for c in rounded], max(abs(error(rounded, f)) for f in grid)


def main() -> None:
    ln2 = mp.log(2)
    ln2_hi = mp.nint(mp.ldexp(ln2, 43)) / mp.mpf(2) ** 43
    ln2_lo = ln2 - ln2_hi
    out = []
    out.append("// Generated by gen_tables.py -- do not edit by hand.")
    out.append("#pragma once")
    out.append("#define CRM_EXP_TABLE_BITS 7")
    out.append("#define CRM_LN2_HI %s" % float.hex(rn(ln2_hi)))
    out.append("#define CRM_LN2_LO %s" % float.hex(rn(ln2_lo)))
    out.append("#define CRM_EXP_TAB_INIT { \\")
    t = exp_table()
    for i in range(0, len(t), 4):
        out.append("    " + ", ".join("0x%016xULL" % v for v in t[i:i + 4]) + ", \\")
    out.append("}")
    rows = log_table()
    for name, col, suffix in (("CRM_LOG_INVC_INIT", 0, "f"), ("CRM_LOG_HI_INIT", 1, ""), ("CRM_LOG_LO_INIT", 2, "f")):
        out.append("#define %s { \\" % name)
        for i in range(0, 128, 4):
            out.append("    " + ", ".join(float.hex(r[col]) + suffix for r in rows[i:i + 4]) + ", \\")
        out.append("}")
    for degree in (5, 6):
        coefficients, error = exp2_poly(degree)
        out.append("// 2^f, |f| <= 1/2: 1 + C1 f + ... of degree %d, relative error %s" % (degree, mp.nstr(error, 3)))
        for i, c in enumerate(coefficients):
            out.append("#define CRM_EXP2_%d_C%d %sf" % (degree, i + 1, float.hex(c)))
    with open(os.path.join(HERE, "crmath_tables.h"), "w") as f:
        f.write("\n".join(out) + "\n")


if __name__ == "__main__":
    main()
