"""The polynomial of the cross attention's exponentials (csrc/cross_attention_tc.cu, exp2_pair) against its generator,
and the error that the kernel's comment states."""
from __future__ import annotations

import pathlib
import re

import numpy as np

from pymsst_b200 import exp2_fit


def _kernel_coefficients():
    src = (pathlib.Path(exp2_fit.__file__).parent / "csrc" / "cross_attention_tc.cu").read_text()
    body = src[src.index("void exp2_pair(") : src.index("unpk2(t, u, v);")]
    first = re.search(r"p = pk2\(([\d.]+)f, \1f\)", body).group(1)
    rest = re.findall(r"p = fma2\(p, f, pk2\(([\d.]+)f, \1f\)\)", body)
    assert rest[-1] == "1."
    return np.array([float(v) for v in [first, *rest[:-1]]][::-1], dtype=np.float32)


def test_fit_reproduces_the_kernel_coefficients():
    """1e-5 is the least squares' freedom: the highest term is 4e-5 of the value, so 1e-5 of it is below 2^-30."""
    np.testing.assert_allclose(_kernel_coefficients(), exp2_fit.fit(), rtol=1e-5, atol=0)


def test_error_of_the_kernel_arithmetic():
    coef = _kernel_coefficients()
    assert exp2_fit.largest_error(coef) < 2.0**-22.4
    x = np.array([-np.inf, -1e30, -127.0, -126.6, 0.0, 8.0, -3.0], dtype=np.float32)
    assert exp2_fit.exp2_fp32(x, coef).tolist() == [0.0, 0.0, 0.0, 0.0, 1.0, 256.0, 0.125]
