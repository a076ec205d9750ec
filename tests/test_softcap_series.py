"""The polynomials that the attention's softcap takes for tanh below 1/2, as the source has them: how far they
are from tanh, by themselves and evaluated in fp32."""

import os
import re

import numpy as np
import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pulsar_amd", "csrc",
                      "paged_attention_parts.h")


def _coefficients(name):
    """Of p, the highest power first: the fp32 constants, as numbers in 64 bits."""
    with open(SOURCE) as f:
        body = re.search(rf"float {name}\(float x\) {{(.*?)\n}}", f.read(), re.S).group(1)
    out = []
    for first, other in re.findall(r"float p = ([^;]+);|fmaf\(p, y, ([^)]+)\)", body):
        text = first or other
        if "0x" in text:
            out.append(float.fromhex(text.rstrip("f")))
        else:
            over, under = text.split("/")
            out.append(float(np.float32(float(over.replace("f", ""))) / np.float32(float(under))))
    return out


@pytest.mark.parametrize("name,terms,itself,in_fp32", [("tanh_series", 6, 2.0 ** -23.4, 3.0), ("tanh_fit", 4, 2.0 ** -25.7, 1.25)])
def test_polynomials(name, terms, itself, in_fp32):
    """x + x y p(y) with y = x^2; in_fp32 is in units of 2^-24."""
    coefficients = _coefficients(name)
    assert len(coefficients) == terms
    x = np.linspace(0, 0.5, 200001)[1:]
    y, p = x * x, coefficients[0]
    for c in coefficients[1:]:
        p = p * y + c
    assert np.abs((x * y * p + x) / np.tanh(x) - 1).max() <= itself
    x = x.astype(np.float32)
    y, p = x * x, np.full_like(x, np.float32(coefficients[0]))

    def fma(a, b, c):  # the product is exact in 64 bits
        return (a.astype(np.float64) * b + c).astype(np.float32)

    for c in coefficients[1:]:
        p = fma(p, y, c)
    got = fma(x * y, p, x.astype(np.float64))
    assert np.abs(got / np.tanh(x.astype(np.float64)) - 1).max() <= in_fp32 * 2.0 ** -24
