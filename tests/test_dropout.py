"""Counter-based dropout (elementwise forms) against its 64-bit definition, and its refusals."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import context_ref as ref
from pymsst_b200 import _native as nat
from pymsst_b200.cross_attention import cross_attention
from pymsst_b200.dropout import DropoutGenerator, drop_threshold, dropout, gelu_dropout

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _key(seed, step, device):
    return torch.tensor([seed, step], dtype=torch.int64, device=device)


# ------------------------------------------------------------------ definition (CPU)
def test_bits_are_uniform_and_tell_sites_and_steps_apart():
    """Over 2^18 numbers a fair 16-bit mean is off by at most 6 sigma, sigma = 65536 / sqrt(12 n); two streams agree
    in an element with probability 2^-16, so in fewer than 40 of 2^18 places (mean 4)."""
    g = np.arange(2**15, dtype=np.uint64)
    base = ref.philox16(g, 0, 0xFFFFFFFF, 5, 9, 2).reshape(-1)
    n = base.size
    assert abs(base.mean() - 65535 / 2) < 6 * 65536 / np.sqrt(12 * n)
    for seed, step, site in ((6, 9, 2), (5, 10, 2), (5, 9, 3), (5 + (1 << 40), 9, 2)):
        other = ref.philox16(g, 0, 0xFFFFFFFF, seed, step, site).reshape(-1)
        assert (base == other).sum() < 40


# Philox4x32 with seven rounds, the known answers that its authors published with it: counter words, key words, result
# words.
KNOWN = [
    ((0, 0, 0, 0), (0, 0), (0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0x4DFCCABA, 0x190A87F0, 0xC47362BA, 0xB6B5242A)),
]


@pytest.mark.parametrize("counter,key,words", KNOWN)
def test_bits_are_the_published_generators(counter, key, words):
    got = ref.philox16(*counter[:3], key[0] | (key[1] << 32), counter[3], 0).tolist()
    assert got == [half for w in words for half in (w & 0xFFFF, w >> 16)]


def test_multiplier_keeps_the_mean():
    mult = ref.dropout_mult(2**18, 0.1, 3, 0, 0)
    t, c = ref.drop_scale(0.1)
    kept = 1 - t / 65536
    # the kept count is binomial: 6 sigma
    assert abs(float(mult.mean()) - 1.0) < 6 * c * np.sqrt(kept * (1 - kept) / 2**18)


@pytest.mark.parametrize("p", [-0.1, 1.5, float("nan")])
def test_probability_outside_the_range_is_refused(p):
    with pytest.raises(ValueError):
        drop_threshold(p)


def test_refusals_on_cpu():
    x = torch.randn(4, 8)
    key = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(nat.FusedKernelUnavailable):
        dropout(x, 0.5, key)
    with pytest.raises(nat.FusedKernelUnavailable):
        gelu_dropout(x, 0.5, key)
    with pytest.raises(ValueError, match="needs a key"):
        dropout(x, 0.5)
    with pytest.raises(ValueError, match="key must be"):
        dropout(x, 0.5, key.int())
    with pytest.raises(ValueError, match="key must be"):
        gelu_dropout(x, 0.5, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="site"):
        dropout(x, 0.5, key, site=-1)
    with pytest.raises(ValueError, match="residual"):
        dropout(x, 0.5, key, residual=torch.zeros(8))
    with pytest.raises(ValueError, match="residual"):
        dropout(x, 0.5, key, residual=x.double())


def test_c_entries_refuse_bad_arguments_without_a_gpu():
    lib = nat.library()
    assert lib.pmb_dropout(None, None, None, -1, 0, None, 0, 0, None) == -1
    assert lib.pmb_dropout(None, None, None, 8, 0, None, 0, 0, None) == -1
    assert lib.pmb_dropout(1, None, 1, 8, 70000, None, 0, 0, None) == -1
    assert b"threshold" in lib.pmb_last_error()
    assert lib.pmb_dropout(16, None, 16, 8, 10, None, 0, 0, None) == -1
    assert b"NULL key" in lib.pmb_last_error()
    assert lib.pmb_dropout(16, None, 16, 8, 0, None, 0, 9, None) == -2
    assert lib.pmb_gelu_dropout_backward(None, 16, 16, 8, 0, None, 0, 0, None) == -1
    assert lib.pmb_dropout_next_key(None, None, None) == -1
    assert lib.pmb_dropout(None, None, None, 0, 0, None, 0, 0, None) == 0


# ------------------------------------------------------------------ kernels
def _bound(dtype, exact, magnitude):
    """One rounding to dtype, and three fp32 roundings (the scale, the product, the sum) of the terms."""
    u = torch.finfo(dtype).eps / 2
    return u * exact.abs() + torch.finfo(dtype).smallest_normal * u + 3 * 2.0**-24 * magnitude


def _close(got, exact, bound):
    err = (got.double().cpu() - exact).abs()
    assert bool((err <= bound).all()), f"off by {float((err / bound.clamp_min(1e-300)).max()):.3f} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,p", [(1, 0.5), (7, 0.3), (8, 0.3), (9, 0.9), (4099, 0.1), (300_001, 0.25), (1 << 21, 0.1),
                                 (1000, 0.0), (1000, 1.0), (0, 0.3)])
def test_dropout_with_and_without_residual(cuda_device, dtype, n, p):
    g = torch.Generator().manual_seed(n + 1)
    x, r, gy = (torch.randn(n, generator=g).to(dtype) for _ in range(3))
    seed, step, site = 0x1234_5678_9ABC_DEF0 >> 1, 2**32 + 5, 2**32 - 1
    mult = ref.dropout_mult(n, p, seed, step, site)
    key = _key(seed, step, cuda_device)
    xd, rd = (t.to(cuda_device).requires_grad_() for t in (x, r))
    y = dropout(xd, p, key, site)
    exact = x.double() * mult
    _close(y.detach(), exact, _bound(dtype, exact, exact.abs()))
    (gx,) = torch.autograd.grad(y, xd, gy.to(cuda_device))
    exact_g = gy.double() * mult
    _close(gx, exact_g, _bound(dtype, exact_g, exact_g.abs()))
    assert bool((gx.cpu()[mult == 0] == 0).all())
    y = dropout(xd, p, key, site, residual=rd)
    exact = x.double() * mult + r.double()
    _close(y.detach(), exact, _bound(dtype, exact, (x.double() * mult).abs() + r.double().abs()))
    gx2, gr = torch.autograd.grad(y, (xd, rd), gy.to(cuda_device))
    assert torch.equal(gx, gx2) and torch.equal(gr.cpu(), gy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,p", [(1, 1, 0.5), (3, 5, 0.2), (62, 768, 0.1), (129, 250, 0.5), (2000, 768, 0.0)])
def test_gelu_dropout(cuda_device, dtype, rows, cols, p):
    """16-bit types: the GELU's fitted exponent leaves a relative error below 2^-14 (exhaustively under one unit of
    fp16, 2^-10); fp32: erff within a few units of the 1 it is added to, so |x| 2^-21 absolute.
    Below x = -5.5 the package's 16-bit GELU takes Phi as 0, as 1 + erf does in fp32: Phi(-5.5) = 1.9e-8 < 2^-25, so
    at most |x| 2^-25 (times the scale) is missing there, and 2^-25 |gy| of the gradient."""
    g = torch.Generator().manual_seed(rows)
    x, gy = ((3 * torch.randn(rows, cols, generator=g)).to(dtype) for _ in range(2))
    seed, step, site = -3, 17, 4
    mult = ref.dropout_mult(rows * cols, p, seed, step, site).reshape(rows, cols)
    key = _key(seed, step, cuda_device)
    xd = x.to(cuda_device).requires_grad_()
    y = gelu_dropout(xd, p, key, site)
    (gx,) = torch.autograd.grad(y, xd, gy.to(cuda_device))
    x64 = x.double()
    cdf = 0.5 * torch.erfc(-x64 * 2.0**-0.5)
    pdf = torch.exp(-0.5 * x64 * x64) / np.sqrt(2 * np.pi)
    exact = mult * x64 * cdf
    exact_g = mult * gy.double() * (cdf + x64 * pdf)
    if dtype == torch.float32:
        slack = mult * x64.abs() * 2.0**-21
        slack_g = mult * gy.double().abs() * (1 + x64.abs()) * 2.0**-21
    else:
        slack = 2.0**-14 * exact.abs() + mult * (x64 < -5.5) * x64.abs() * 2.0**-25
        slack_g = mult * gy.double().abs() * (2.0**-14 * (cdf + (x64 * pdf).abs()) + (x64 < -5.5) * 2.0**-25)
    _close(y.detach(), exact, _bound(dtype, exact, exact.abs()) + slack)
    _close(gx, exact_g, _bound(dtype, exact_g, exact_g.abs()) + slack_g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_kernel_bits_are_the_published_generators(cuda_device, dtype):
    """Eight keys of the first query, head and batch item, seed, step and site 0: the zero counter under the zero key.
    Each of its eight numbers u keeps its key at a threshold of u and drops it at u + 1.  Scores of zero and the
    identity as values show the kept ones."""
    words = KNOWN[0][2]
    numbers = [half for w in words for half in (w & 0xFFFF, w >> 16)]
    q, k = torch.zeros(1, 1, 1, 8, device=cuda_device, dtype=dtype), torch.zeros(1, 1, 8, 8, device=cuda_device, dtype=dtype)
    v = torch.eye(8, device=cuda_device, dtype=dtype).reshape(1, 1, 8, 8)
    key = _key(0, 0, cuda_device)
    for u in numbers:
        for threshold in (u, u + 1):
            o = cross_attention(q, k, v, dropout_p=threshold / 65536, key=key)
            assert (o.flatten() != 0).tolist() == [n >= threshold for n in numbers]


@pytest.mark.gpu
def test_unaligned_and_strided_inputs(cuda_device):
    """Elements are numbered by the logical index: views give what their contiguous copies give."""
    key = _key(1, 2, cuda_device)
    base = torch.randn(40, 33, device=cuda_device, dtype=torch.bfloat16)
    for view in (base[1:, :], base.t(), base[:, 1:30], base.reshape(-1)[3:1000], base[::2, ::3]):
        assert torch.equal(dropout(view, 0.3, key, 1), dropout(view.clone(), 0.3, key, 1))
        assert torch.equal(gelu_dropout(view, 0.3, key, 1), gelu_dropout(view.clone(), 0.3, key, 1))
        res = torch.randn_like(view)
        assert torch.equal(dropout(view, 0.3, key, 1, residual=res), dropout(view.clone(), 0.3, key, 1, residual=res))
    x = torch.randn(8, 16, device=cuda_device, requires_grad=True)
    y = dropout(x, 0.5, key)
    (g1,) = torch.autograd.grad(y, x, torch.ones(1, 1, device=cuda_device).expand(8, 16), retain_graph=True)
    (g2,) = torch.autograd.grad(y, x, torch.ones(8, 16, device=cuda_device))
    assert torch.equal(g1, g2)


@pytest.mark.gpu
def test_dropped_values_never_reach_the_result(cuda_device):
    key = _key(11, 0, cuda_device)
    n = 4096
    mult = ref.dropout_mult(n, 0.4, 11, 0, 0)
    x = torch.ones(n)
    x[mult == 0] = torch.nan
    for dtype in TYPES:
        xd = x.to(dtype).to(cuda_device)
        for y in (dropout(xd, 0.4, key), gelu_dropout(xd, 0.4, key), dropout(xd, 0.4, key, residual=torch.ones_like(xd))):
            assert bool(torch.isfinite(y).all())
        assert bool((dropout(xd, 1.0, key) == 0).all())


@pytest.mark.gpu
def test_broadcast_input_and_residual_gradients(cuda_device):
    key = _key(5, 5, cuda_device)
    x = torch.randn(1, 16, device=cuda_device, requires_grad=True)
    y = dropout(x.expand(24, 16), 0.25, key, 3, residual=x.expand(24, 16))
    gy = torch.randn(24, 16, device=cuda_device)
    (gx,) = torch.autograd.grad(y, x, gy)
    mult = ref.dropout_mult(24 * 16, 0.25, 5, 5, 3).reshape(24, 16)
    exact = (gy.double().cpu() * (mult + 1)).sum(0, keepdim=True)
    # 25 fp32 additions of each column
    assert torch.allclose(gx.double().cpu(), exact, rtol=0, atol=30 * 2.0**-24 * float(
        (gy.double().cpu().abs() * (mult + 1)).sum(0).max()))


@pytest.mark.gpu
def test_key_changed_before_the_backward_is_an_error(cuda_device):
    key = _key(1, 1, cuda_device)
    x = torch.randn(64, device=cuda_device, requires_grad=True)
    y = dropout(x, 0.5, key)
    key.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.gpu
def test_second_derivatives_are_refused(cuda_device):
    x = torch.randn(64, device=cuda_device, requires_grad=True)
    y = gelu_dropout(x, 0.5, _key(1, 1, cuda_device))
    (g,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice"):
        g.sum().backward()


@pytest.mark.gpu
def test_generator_state_used_as_key_is_an_error_after_its_next_key(cuda_device):
    gen = DropoutGenerator(5, cuda_device)
    x = torch.randn(64, device=cuda_device, requires_grad=True)
    y = dropout(x, 0.5, gen.state)
    gen.next_key()
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.gpu
def test_generator_steps_and_restores(cuda_device):
    gen = DropoutGenerator(2**64 - 2, cuda_device)
    k0, k1 = gen.next_key(), gen.next_key()
    assert k0.tolist() == [-2, 0] and k1.tolist() == [-2, 1]
    state = gen.state_dict()
    x = torch.randn(1000, device=cuda_device)
    a = dropout(x, 0.5, gen.next_key())
    gen.load_state_dict(state)
    assert torch.equal(a, dropout(x, 0.5, gen.next_key()))
    assert not torch.equal(a, dropout(x, 0.5, gen.next_key()))


@pytest.mark.gpu
def test_captured_forward_draws_new_masks_and_its_backward_matches(cuda_device):
    gen = DropoutGenerator(7, cuda_device)
    x = torch.ones(1 << 14, device=cuda_device, requires_grad=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = dropout(x, 0.5, gen.next_key(), 2)
        torch.autograd.grad(y.sum(), x)
        del y
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dropout(x, 0.5, gen.next_key(), 2)
        (gx,) = torch.autograd.grad(y.sum(), x)
        y = y.detach()
    seen = []
    for replay in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, gx)  # x is one, dL/dy is one
        mult = ref.dropout_mult(x.numel(), 0.5, 7, 1 + replay, 2)
        assert torch.equal(y.cpu().double(), mult)
        seen.append(y.clone())
    assert not torch.equal(seen[0], seen[1])
