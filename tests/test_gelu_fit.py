"""The polynomial of the GELU epilogue (csrc/fd_w8a8.h), read from its source and evaluated on the CPU against math.erfc.

The fit's own error is stated there as 9e-8. With u = 2^-24, float32's half step, Horner's eight steps of two roundings are
off by at most 16 u sum |c_i| t^i, and that sum is at most 2.16 P(t) (checked below): 35 u of P. t carries three
roundings, in t and, with t P' / P <= 1.26, in P, and three products and the exponential's own step follow:
35 u + 7 u + 4 u + the fit's 2 u < 64 u = 2^-18. The exponential's argument carries the square's rounding, log2(e)'s and the
product's, 3 u of v^2 / 2, below 2^-22 of it."""

from __future__ import annotations

import math
import re
from pathlib import Path

import numpy as np

SOURCE = Path(__file__).resolve().parents[1] / "fused-decode_amd" / "csrc" / "fd_w8a8.h"


def coefficients():
    body = SOURCE.read_text().split("float gelu(float v) {")[1].split("const float tail")[0]
    first = re.search(r"float p = (-?[\d.]+)f;", body).group(1)
    rest = re.findall(r"p = p \* t ([+-]) ([\d.]+)f;", body)
    slope = re.search(r"1\.f \+ ([\d.]+)f \* a", body).group(1)
    return [float(first)] + [float(s + c) for s, c in rest], float(slope)


def test_the_fit():
    c, slope = coefficients()
    assert len(c) == 9 and abs(slope - 8**-0.5) < 2.0**-25
    c = [float(np.float32(v)) for v in c]
    for i in range(1001):
        t = i / 1000
        terms = [v * t**k for k, v in enumerate(reversed(c))]
        slopes = [k * term for k, term in enumerate(terms)]
        assert sum(map(abs, terms)) <= 2.16 * sum(terms) and abs(sum(slopes)) <= 1.26 * sum(terms)
    worst = 0.0
    for i in range(1, 13001):
        z = i / 1000
        t, p = 1 / (1 + z * math.sqrt(2) * float(np.float32(slope))), 0.0
        for v in c:
            p = p * t + v
        worst = max(worst, abs(p * 2 * t / (math.exp(z * z) * math.erfc(z)) - 1))
    assert worst < 9e-8


def test_its_evaluation_in_float32():
    c, slope = coefficients()
    f = np.float32
    v = np.concatenate([np.linspace(-9, 9, 40001), [-1e-3, 1e-3, 0.0]]).astype(f)
    a = np.abs(v)
    t = f(1) / (f(1) + f(slope) * a)
    p = np.full_like(t, f(c[0]))
    for k in c[1:]:
        p = p * t + f(k)
    tail = a * (np.exp2((f(-0.5) * a * a) * f(math.log2(math.e))) * t * p)
    y = np.where(v < 0, -tail, v - tail).astype(np.float64)
    want = np.array([0.5 * float(x) * math.erfc(-float(x) / math.sqrt(2)) for x in v])
    bound = (2.0**-18 + 2.0**-22 * v.astype(np.float64) ** 2 / 2) * np.abs(want) + 2.0**-126
    assert (np.abs(y - want) <= bound).all()
