"""The polynomial that computes some of the exponentials of packed attention on the FMA pipe, evaluated with the coefficients of the source."""
import os
import re

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_polynomial_of_the_exponentials():
    """2^f on [-1/2, 1/2] within the 3.6e-6 that the source says, with each step rounded to fp32, and 1 at 0."""
    source = open(os.path.join(ROOT, "cuda-kernel-qwen3-8b-awq_b200", "csrc", "attn_packed_tc.cu")).read()
    body = source[source.index("float2 pk_ex2_fma("):]
    body = body[:body.index("return")]
    first = re.search(r"fma2\(make_float2\(([\d.]+)f, \1f\), f, make_float2\(([\d.]+)f, \2f\)\)", body)
    rest = re.findall(r"p = fma2\(p, f, make_float2\(([\d.]+)f, \1f\)\)", body)
    coefficients = [np.float32(x) for x in (*first.groups(), *rest)]
    assert len(coefficients) == 5 and coefficients[-1] == 1
    f = np.linspace(-0.5, 0.5, 200001).astype(np.float32)
    p = np.full_like(f, coefficients[0])
    for c in coefficients[1:]:
        p = (p.astype(np.float64) * f + c).astype(np.float32)      # a product and a sum, rounded once: exact in 64 bits beforehand, but for a double rounding
    assert p[100000] == 1 and np.abs(p / np.exp2(f.astype(np.float64)) - 1).max() <= 3.6e-6 + 2.0 ** -23
