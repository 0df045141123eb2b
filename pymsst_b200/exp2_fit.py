"""Coefficients of the 2^f polynomial that takes part of the cross attention's exponentials off the special-function pipe
(csrc/cross_attention_tc.cu, exp2_pair).

2^x = 2^n 2^f with n the integer nearest to x (range reduction as in Cody and Waite, Software Manual for the Elementary
Functions, 1980).  2^f on [-1/2, 1/2] is a degree-five polynomial with the constant term fixed at 1, so that 2^0 is
exact, fitted by least squares of the relative error on a Chebyshev grid with the weights raised where the error is
largest (Lawson's iteration toward the minimax fit), keeping the iterate whose largest error is smallest.

``python -m pymsst_b200.exp2_fit`` prints the coefficients and the largest relative error of an fp32 emulation of the
kernel arithmetic.  The library itself does not import this module.
"""
from __future__ import annotations

import numpy as np

DEGREE = 5


def fit(degree: int = DEGREE, nodes: int = 8001, iterations: int = 400) -> np.ndarray:
    """fp32 coefficients of f, f^2, ... f^degree."""
    f = 0.5 * np.cos(np.linspace(0, np.pi, nodes))
    f = f[np.abs(f) > 1e-9]
    y = 2.0**f
    a, b = np.vander(f, degree + 1, increasing=True)[:, 1:] / y[:, None], 1 - 1 / y
    w = np.ones_like(f)
    best, coef = np.inf, None
    for _ in range(iterations):
        c, *_ = np.linalg.lstsq(a * np.sqrt(w)[:, None], b * np.sqrt(w), rcond=None)
        err = np.abs(a @ c - b)
        if err.max() < best:
            best, coef = err.max(), c
        w = w * (err / err.max() + 1e-3) ** 0.5
        w /= w.mean()
    return coef.astype(np.float32)


def exp2_fp32(x: np.ndarray, coef: np.ndarray) -> np.ndarray:
    """fp32 emulation of the kernel's 2^x for x <= 127 (a fused multiply-add is one rounding of the exact result)."""
    x = np.maximum(x.astype(np.float32), np.float32(-127))
    t = x + np.float32(12582912)
    f = x - (t - np.float32(12582912))
    p = np.full_like(f, coef[-1])
    for c in [*coef[-2::-1], np.float32(1)]:
        p = (p.astype(np.float64) * f + c).astype(np.float32)
    bits = (t.view(np.int32).astype(np.int64) << 23) + 0x3F800000
    return p * (bits & 0xFFFFFFFF).astype(np.uint32).view(np.float32)


def largest_error(coef: np.ndarray, count: int = 4_000_001) -> float:
    """Largest relative error over [-125.5, 8], where the results are normal numbers."""
    x = np.linspace(-125.5, 8, count).astype(np.float32)
    return float(np.abs(exp2_fp32(x, coef).astype(np.float64) / 2.0 ** x.astype(np.float64) - 1).max())


def main() -> None:
    coef = fit()
    print(", ".join("%.16gf" % c for c in coef))
    print("largest relative error: 2^%.2f" % np.log2(largest_error(coef)))


if __name__ == "__main__":
    main()
