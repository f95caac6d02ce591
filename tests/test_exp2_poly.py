"""The powers of two that the attention of many rows takes on the multipliers (ex2_poly in rows_attn_tc.cu), computed here as the kernel does, with the coefficients
of its source, against 64 bits (no GPU)."""
import os
import re

import numpy as np

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "asrq_b200", "csrc", "rows_attn_tc.cu")


def _coefficients():
    with open(SOURCE) as f:
        body = f.read().split("ex2_poly(unsigned long long x) {", 1)[1].split("\n}\n", 1)[0]
    assert "12582912.f + 127.f" in body
    found = dict(re.findall(r"\b(c[0-4]) = ([0-9.e-]+)f", body))
    return [np.float32(found[f"c{i}"]) for i in range(5)]


def _fma(a, b, c):  # one rounding to 32 bits: a product of two of them is exact in 64
    return (a.astype(np.float64) * b.astype(np.float64) + np.float64(c)).astype(np.float32)


def _ex2(x):
    c = _coefficients()
    shift = np.float32(12582912.0 + 127.0)
    x = np.maximum(x.astype(np.float32), np.float32(-126))
    i = x + shift
    f = x - (i - shift)  # exact
    assert f.dtype == np.float32 and float(np.abs(f).max()) <= 0.5
    y = _fma(np.full_like(f, c[4]), f, c[3])
    for k in (2, 1, 0):
        y = _fma(y, f, c[k])
    exponent = (i.view(np.uint32) << np.uint32(23)).view(np.float32)  # the low bits: whole part and the exponent's bias
    return (y * exponent).astype(np.float32)


def test_within_its_error():
    """2.6e-6 relative for the polynomial, 5 roundings of 2^-24."""
    for lo, hi, n in ((-0.5, 0.5, 400001), (-126, 16, 2000001), (-30, 0, 500001)):
        x = np.linspace(lo, hi, n).astype(np.float32)
        want = np.exp2(x.astype(np.float64))
        off = np.abs(_ex2(x).astype(np.float64) - want) / want
        assert off.max() <= 2.6e-6 + 5 * 2.0 ** -24, (lo, hi, off.max())


def test_at_whole_numbers_and_far_below():
    x = np.arange(-126, 101).astype(np.float32)
    assert np.abs(_ex2(x).astype(np.float64) / np.exp2(x.astype(np.float64)) - 1).max() <= 2.6e-6
    assert (_ex2(np.array([-127.0, -1e4, -3e38, -np.inf], dtype=np.float32)) <= 2.0 ** -125.9).all()
