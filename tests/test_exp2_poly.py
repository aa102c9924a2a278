"""CPU check of the FMA-pipe exp2 in csrc/fa_fwd_kernel.cuh (`exp2_poly2`).

The kernel can route a share of its exp2s through a polynomial instead of `ex2.approx`
(`FA_POLY_PAIRS_OF_8`).  This test replays the routine's exact fp32 / bit steps in numpy --
clamp, round-to-integer by adding 1.5 * 2^23, f = x - n, degree-4 Horner with fused
multiply-adds, and n added to the exponent field -- using the constants read from the kernel
source, and checks the result against exp2 over the whole range a softmax step can produce
(masked logits are -inf).  A clamp one lower (-127) would let 2^f < 1 borrow through the
exponent field into the sign bit, giving a NaN pattern; the test shows that too.
"""
from __future__ import annotations

import re
from pathlib import Path

import numpy as np

KERNEL = Path(__file__).resolve().parents[1] / "flash_attn_npu_b200" / "csrc" / "fa_fwd_kernel.cuh"


def _constants():
    src = KERNEL.read_text()
    body = src[src.index("float2 exp2_poly2(float2 x)"):]
    body = body[:body.index("return q;")]
    coeffs = [float(m) for m in re.findall(r"c\d = ([-+0-9.eE]+)f", body)]
    clamp = float(re.search(r"fmaxf\(x\.x, (-[0-9.]+)f\)", body).group(1))
    assert len(coeffs) == 5
    return np.array(coeffs, dtype=np.float32), np.float32(clamp)


def _fma(a, b, c):
    # fp32 fused multiply-add: exact product in fp64, one rounding of the sum to fp32
    return (a.astype(np.float64) * b.astype(np.float64) + c.astype(np.float64)).astype(np.float32)


def exp2_poly_emulated(x, coeffs, clamp):
    x = np.maximum(np.asarray(x, dtype=np.float32), clamp)
    r = np.float32(12582912.0)  # 1.5 * 2^23
    t = (x + r).astype(np.float32)
    n = (t - r).astype(np.float32)
    f = _fma(n, np.full_like(n, -1.0), x)
    c0, c1, c2, c3, c4 = (np.full_like(f, c) for c in coeffs)
    q = _fma(c4, f, c3)
    q = _fma(q, f, c2)
    q = _fma(q, f, c1)
    q = _fma(q, f, c0)
    bits = q.view(np.uint32) + (t.view(np.uint32) << np.uint32(23))
    return bits.astype(np.uint32).view(np.float32)


def test_exp2_poly_matches_exp2_over_the_softmax_range():
    coeffs, clamp = _constants()
    x = np.concatenate([np.linspace(-300.0, 8.0, 400001, dtype=np.float32),
                        np.array([-np.inf, -127.0, -126.5, -126.0, -125.5, 0.0, 8.0],
                                 dtype=np.float32)])
    with np.errstate(invalid="ignore", over="ignore"):
        y = exp2_poly_emulated(x, coeffs, clamp)
    assert np.all(np.isfinite(y)) and np.all(y >= 0.0)
    ref = np.exp2(x.astype(np.float64))
    normal = x >= -125.0
    rel = np.abs(y[normal].astype(np.float64) / ref[normal] - 1.0)
    assert rel.max() < 3e-6, rel.max()
    # below 2^-125 the result is only required to be tiny and non-negative
    assert np.all(y[~normal] <= 2.0 ** -124)


def test_clamp_one_lower_would_produce_nan():
    coeffs, _ = _constants()
    with np.errstate(invalid="ignore"):
        y = exp2_poly_emulated(np.array([-127.0, -126.6], dtype=np.float32), coeffs,
                               np.float32(-127.0))
    assert np.isnan(y[0]) or y[0] < 0.0


# ------------------------------------------------ add_exp2_poly of fa_paged_weights.cuh, the same way
WEIGHTS = KERNEL.with_name("fa_paged_weights.cuh")


def add_exp2_poly_emulated(x):
    """0 + 2^x in the routine's steps, with the constants of its source."""
    src = WEIGHTS.read_text()
    body = src[src.index("float2 add_exp2_poly("):]
    body = body[:body.index("\n}\n")]
    coeffs = [np.float32(m) for m in re.findall(r"c\d = ([-+0-9.eE]+)f", body)]
    assert len(coeffs) == 6
    lo, hi = (np.array([int(m, 16)], np.uint32).view(np.float32)[0] for m in re.findall(r"0f([0-9A-F]{8})", body))
    exponent = {int(m, 16) for m in re.findall(r"<< 23\) \+ (0x[0-9a-f]+)\)", body)}
    assert len(exponent) == 1
    x = np.asarray(x, dtype=np.float32)
    x = np.where(np.isnan(x), x, np.minimum(np.maximum(x, lo), hi))
    r = np.float32(12582912.0)
    t = (x + r).astype(np.float32)
    f = _fma((t - r).astype(np.float32), np.full_like(x, -1.0), x)
    q = np.full_like(f, coeffs[-1])
    for c in coeffs[-2::-1]:
        q = _fma(q, f, np.full_like(f, c))
    scale = ((t.view(np.uint32) << np.uint32(23)) + np.uint32(exponent.pop())).view(np.float32)
    return _fma(q, scale, np.zeros_like(q))


def test_add_exp2_poly_is_exp2_as_far_as_fp32_goes():
    """Relative error 2.4e-7 (the fit's) up to the largest finite power, infinite from 128, 0 at the far end."""
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.concatenate([np.linspace(-125.5, 128.0, 400001, dtype=np.float32)[1:-1],
                            np.nextafter(np.float32([127.5, 128, -125, 0.5, -0.5]), np.float32(-200)),
                            np.float32([127.5, 127.75, 127.9, 0, 1, -1])])
        x = x[x < 128]
        y = add_exp2_poly_emulated(x).astype(np.float64)
        # (exp2 of what the largest x is, to fp32, may round up to infinity)
        near = x > 127.99999
        assert np.all(np.isfinite(y[~near])) and np.all(y > 0)
        assert np.abs(y[~near] / np.exp2(x[~near].astype(np.float64)) - 1).max() < 2.4e-7
        assert np.all(add_exp2_poly_emulated([128.0, 129.0, 3e38, np.inf]) == np.inf)
        assert np.all(add_exp2_poly_emulated([-126.51, -127.0, -200.0, -3e38, -np.inf]) == 0.0)
        low = add_exp2_poly_emulated(np.linspace(-126.5, -125.5, 1001, dtype=np.float32))
        assert np.all((low >= 0) & (low <= 2.0 ** -125.49))
        assert np.isnan(add_exp2_poly_emulated([np.nan]))[0]


def test_coefficients_are_those_of_the_fit():
    import importlib.util
    spec = importlib.util.spec_from_file_location("exp2_poly_fit", KERNEL.with_name("exp2_poly_fit.py"))
    fit = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(fit)
    src = WEIGHTS.read_text()
    body = src[src.index("float2 add_exp2_poly("):]
    coeffs = np.float32(re.findall(r"c\d = ([-+0-9.eE]+)f", body[:body.index("return ffma2")]))
    assert np.allclose(coeffs / np.round(coeffs[0]), fit.fit(5), rtol=2.0 ** -22, atol=0)
