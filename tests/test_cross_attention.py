"""Cross attention (padded keys, shared heads, dropout on the probabilities) against the 64-bit definition."""
from __future__ import annotations

import pytest
import torch

from oracle import context_ref as ref
from pymsst_b200 import _native as nat
from pymsst_b200.cross_attention import cross_attention

SEED, STEP, SITE = 0x0BAD_5EED_1234_5678, 41, 6


def _key(device):
    return torch.tensor([SEED, STEP], dtype=torch.int64, device=device)


def _inputs(b, hq, hk, nq, nk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(1000 + seed + 7 * nq + nk)
    q = torch.randn(b, nq, hq, d, generator=g).to(dtype).transpose(1, 2)
    k, v = (torch.randn(b, nk, hk, d, generator=g).to(dtype).transpose(1, 2) for _ in range(2))
    go = torch.randn(b, nq, hq, d, generator=g).to(dtype).transpose(1, 2)
    return q, k, v, go


def _mult(q, k, p):
    if p == 0:
        return None
    return ref.attention_mult(q.shape[0], q.shape[1], q.shape[2], k.shape[2], p, SEED, STEP, SITE)


def _within(got, exact, bound, what):
    err = (got.detach().double().cpu() - exact).abs()
    worst = float((err / bound.clamp_min(1e-300)).max()) if err.numel() else 0.0
    assert bool((err <= bound).all()), f"{what}: off by {worst:.3f} of the bound"


def _splits(b, hq, hk, nq, nk, d, dtype):
    """Whether the forward of this shape joins several key ranges."""
    return nat.library().pmb_cross_attention_forward_workspace_size(b, hq, hk, nq, nk, d, nat.dtype_code(dtype)) > 0


def _check(device, q, k, v, go, lengths=None, p=0.0, scale=None, lengths_dtype=torch.int32):
    dtype = q.dtype
    leaves = [t.to(device).requires_grad_() for t in (q, k, v)]
    dev_len = None if lengths is None else torch.tensor(lengths, dtype=lengths_dtype, device=device)
    key = _key(device) if p > 0 else None
    o = cross_attention(*leaves, key_lengths=dev_len, scale=scale, dropout_p=p, key=key, site=SITE)
    grads = torch.autograd.grad(o, leaves, go.to(device))
    with torch.no_grad():
        again = cross_attention(*leaves, key_lengths=dev_len, scale=scale, dropout_p=p, key=key, site=SITE)
    assert torch.equal(again, o.detach())
    q64, k64, v64, g64 = (t.double() for t in (q, k, v, go))
    mult = _mult(q, k, p)
    exact = (ref.attention(q64, k64, v64, lengths, scale, mult),
             *ref.attention_grads(q64, k64, v64, g64, lengths, scale, mult))
    bounds = ref.attention_bounds(q64, k64, v64, g64, lengths, scale, mult, dtype)
    for got, e, bound, what in zip((o, *grads), exact, bounds, ("o", "dq", "dk", "dv")):
        assert got.shape == e.shape and got.dtype == dtype
        _within(got, e, bound, what)
    assert int(nat.library().pmb_umma_timeout(0)) == 0
    return o, grads


# ------------------------------------------------------------------ definition (CPU)
def test_formula_gradients_match_differences():
    """gradcheck: the definition's derivatives against central differences in 64 bits; then the formulas the kernels
    follow against those derivatives."""
    torch.manual_seed(3)
    q = torch.randn(2, 4, 3, 5, dtype=torch.float64, requires_grad=True)
    k, v = (torch.randn(2, 2, 6, 5, dtype=torch.float64, requires_grad=True) for _ in range(2))
    lengths, mult = [4, 0], ref.attention_mult(2, 4, 3, 6, 0.3, SEED, STEP, SITE)
    assert torch.autograd.gradcheck(lambda *a: ref.attention(*a, lengths, 0.7, mult), (q, k, v))
    go = torch.randn(2, 4, 3, 5, dtype=torch.float64)
    auto = torch.autograd.grad(ref.attention(q, k, v, lengths, 0.7, mult), (q, k, v), go)
    with torch.no_grad():
        for a, f in zip(auto, ref.attention_grads(q, k, v, go, lengths, 0.7, mult)):
            assert torch.allclose(a, f, rtol=1e-12, atol=1e-13)
            assert bool((f[1] == 0).all())  # the item without keys


def test_definition_matches_torch():
    torch.manual_seed(4)
    q, k, v = torch.randn(2, 3, 7, 8).double(), torch.randn(2, 3, 9, 8).double(), torch.randn(2, 3, 9, 8).double()
    expect = torch.nn.functional.scaled_dot_product_attention(q, k, v)
    assert torch.allclose(ref.attention(q, k, v), expect, rtol=1e-12, atol=1e-13)


def test_refusals():
    q, k, v, _ = _inputs(2, 4, 2, 3, 5, 8, torch.bfloat16)
    key = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(nat.FusedKernelUnavailable):
        cross_attention(q, k, v)
    for bad in ((q[0], k, v), (q, k, v[:, :, :4]), (q[:1], k, v), (q[..., :4], k, v), (q[:, :3], k, v)):
        with pytest.raises(ValueError):
            cross_attention(*bad)
    with pytest.raises(TypeError):
        cross_attention(q, k.float(), v.float())
    with pytest.raises(TypeError):
        cross_attention(q.double(), k.double(), v.double())
    with pytest.raises(ValueError, match="head dim"):
        cross_attention(*(torch.zeros(1, 1, 2, 257) for _ in range(3)))
    for lengths in (torch.zeros(3, dtype=torch.int32), torch.zeros(2), torch.zeros(2, 1, dtype=torch.int32)):
        with pytest.raises(ValueError, match="key_lengths"):
            cross_attention(q, k, v, key_lengths=lengths)
    with pytest.raises(ValueError, match="needs a key"):
        cross_attention(q, k, v, dropout_p=0.1)
    with pytest.raises(ValueError):
        cross_attention(q, k, v, dropout_p=1.1, key=key)
    with pytest.raises(ValueError, match="site"):
        cross_attention(q, k, v, dropout_p=0.1, key=key, site=2**32)


def test_c_entries_refuse_bad_arguments_without_a_gpu():
    lib = nat.library()
    strides = nat.i64_array([8] * 24)

    def fwd(heads=4, kv=2, dim=8, threshold=0, dtype=2, ptr=16, nq=3):
        return lib.pmb_cross_attention_forward(ptr, ptr, ptr, ptr, ptr, None, 2, heads, kv, nq, 5, dim, strides, 1.0,
                                               threshold, None, 0, dtype, None, 0, None)

    assert fwd(kv=3) == -1 and b"multiple" in lib.pmb_last_error()
    assert fwd(kv=0) == -1 and fwd(dim=0) == -1 and fwd(dim=257) == -1 and fwd(nq=-1) == -1
    assert fwd(threshold=5) == -1 and b"NULL key" in lib.pmb_last_error()
    assert fwd(threshold=-1) == -1 and fwd(ptr=None) == -1
    assert fwd(dtype=7) == -2
    assert lib.pmb_cross_attention_lse_size(2, 4, 3) >= 2 * 4 * 3
    misaligned = nat.i64_array([8, 8, 12] * 8)  # head strides of 12 elements: no 16-byte rows
    assert lib.pmb_cross_attention_forward(16, 16, 16, 16, 16, None, 2, 4, 2, 3, 5, 8, misaligned, 1.0, 0, None, 0, 2,
                                           None, 0, None) == -4
    assert lib.pmb_cross_attention_forward(8, 16, 16, 16, 16, None, 2, 4, 2, 3, 5, 8, strides, 1.0, 0, None, 0, 2,
                                           None, 0, None) == -4
    need = lib.pmb_cross_attention_forward_workspace_size(1, 1, 1, 1, 8192, 64, 2)
    assert need > 0
    assert lib.pmb_cross_attention_forward(16, 16, 16, 16, 16, None, 1, 1, 1, 1, 8192, 64, strides, 1.0, 0, None, 0, 2,
                                           16, need - 1, None) == -5
    size = lib.pmb_cross_attention_backward_workspace_size(2, 4, 2, 3, 5, 8, 2)
    assert size >= 2 * 4 * 3 * 4
    bwd = lib.pmb_cross_attention_backward(16, 16, 16, 16, 16, 16, 16, 16, 16, None, 2, 4, 2, 3, 5, 8, strides, 1.0, 0,
                                           None, 0, 2, 16, size - 1, None)
    assert bwd == -5


def test_c_entries_refuse_sizes_beyond_their_indices_without_a_gpu():
    """Sizes whose 32-bit forms or products would wrap: 0 from the queries, an error from the entries; packed heads of
    many queries stay inside (2^26 queries of 64 heads that share one)."""
    lib = nat.library()
    strides = nat.i64_array([8] * 24)
    packed = (1, 64, 1, 2**26, 1, 8, 2)
    assert lib.pmb_cross_attention_forward_workspace_size(*packed) == 0  # one key range
    assert lib.pmb_cross_attention_backward_workspace_size(*packed) >= 64 * 2**26 * 4
    for sizes in ((1, 2**32, 2**32, 1, 1), (2**32, 1, 1, 1, 1), (2**40, 2**40, 1, 1, 5), (2**15, 2**15, 1, 1, 5),
                  (1, 1, 1, 2**30, 5), (1, 1, 1, 5, 2**32), (1, 2**31, 2**31, 2**31, 5)):
        b, h, hk, nq, nk = sizes
        assert lib.pmb_cross_attention_forward_workspace_size(*sizes, 8, 2) == 0
        assert lib.pmb_cross_attention_backward_workspace_size(*sizes, 8, 2) == 0
        assert nk == 2**32 or lib.pmb_cross_attention_lse_size(b, h, nq) == 0
        assert lib.pmb_cross_attention_forward(16, 16, 16, 16, 16, None, *sizes, 8, strides, 1.0, 0, None, 0, 2, None,
                                               0, None) == -1
        assert b"too large" in lib.pmb_last_error()
        assert lib.pmb_cross_attention_backward(16, 16, 16, 16, 16, 16, 16, 16, 16, None, *sizes, 8, strides, 1.0, 0,
                                                None, 0, 2, None, 0, None) == -1
        assert b"too large" in lib.pmb_last_error()
    one = nat.i64_array([4])
    for batch, tokens, heads in ((2**32, 2**32, 1), (1, 2**32, 2**32), (2**30, 1, 1), (1, 1, 2**62)):
        assert lib.pmb_rotary_axes(16, 16, 16, 16, batch, tokens, heads, 8, strides, 0, 0, 1, one, 0, 2, None) == -1
        assert b"too large" in lib.pmb_last_error()


# ------------------------------------------------------------------ kernels
SHAPES = [
    # b, hq, hk, nq, nk, d
    (1, 1, 1, 1, 1, 8),
    (2, 2, 1, 3, 5, 16),
    (1, 8, 2, 17, 129, 64),
    (2, 4, 4, 128, 64, 64),
    (1, 2, 2, 129, 257, 64),
    (2, 6, 2, 33, 100, 40),
    (1, 3, 1, 70, 300, 128),
    (1, 2, 2, 1, 1000, 64),
    (1, 16, 1, 9, 65, 96),
    (3, 2, 2, 258, 258, 64),
    (1, 4, 2, 300, 31, 72),
    (1, 1, 1, 385, 130, 120),
]


# few row tiles over long contexts: several key ranges, joined by a second kernel
SPLIT = [
    # b, hq, hk, nq, nk, d, lengths
    (3, 8, 2, 5, 3000, 64, None),
    (3, 8, 2, 5, 3000, 64, [0, 100, 3000]),
    (2, 4, 1, 40, 2500, 128, None),
    (2, 4, 1, 40, 2500, 128, [1, 2499]),
    (4, 4, 2, 6, 2500, 96, [0, 1, 100, 2500]),
    (1, 6, 1, 130, 1111, 40, [577]),
    (5, 2, 2, 1, 4001, 8, [4001, 0, 2, 97, 4000]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,p", [(torch.bfloat16, 0.0), (torch.float16, 0.0), (torch.bfloat16, 0.25),
                                     (torch.float16, 0.25)])
@pytest.mark.parametrize("b,hq,hk,nq,nk,d,lengths", SPLIT)
def test_joined_key_ranges_match_the_definition(cuda_device, b, hq, hk, nq, nk, d, lengths, dtype, p):
    """Several rows, batch items, packed heads and head dims through the partial sums and their join, with ranges (and
    whole rows) without keys; NaN and infinities behind the lengths."""
    assert _splits(b, hq, hk, nq, nk, d, dtype)
    q, k, v, go = _inputs(b, hq, hk, nq, nk, d, dtype)
    for i, n in enumerate(lengths or []):
        k[i, :, n:] = torch.nan if i % 2 else torch.inf
        v[i, :, n:] = -torch.inf if i % 2 else torch.nan
    _check(cuda_device, q, k, v, go, lengths, p)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("b,hq,hk,nq,nk,d", SHAPES)
def test_matches_the_definition(cuda_device, b, hq, hk, nq, nk, d, p, dtype):
    _check(cuda_device, *_inputs(b, hq, hk, nq, nk, d, dtype), p=p)


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("b,hq,hk,nq,nk,d", [(1, 1, 1, 1, 1, 1), (2, 4, 2, 37, 70, 64), (1, 2, 1, 5, 33, 256),
                                             (2, 1, 1, 40, 3, 7), (1, 8, 8, 64, 64, 8)])
def test_full_precision(cuda_device, b, hq, hk, nq, nk, d, p):
    _check(cuda_device, *_inputs(b, hq, hk, nq, nk, d, torch.float32), p=p)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [7, 33, 136, 256])
def test_odd_and_wide_heads_in_16_bits(cuda_device, d):
    _check(cuda_device, *_inputs(2, 4, 2, 19, 45, d, torch.bfloat16), p=0.1, lengths=[45, 11])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("nq,nk,p", [(5, 70, 0.0), (130, 200, 0.25), (1, 513, 0.0), (64, 128, 0.1), (258, 385, 0.1)])
def test_key_lengths_with_anything_behind_them(cuda_device, dtype, nq, nk, p):
    """Lengths of nothing, one, odd counts, a tile's border, everything and beyond; NaN and infinities in the padding
    must not reach a result, and its gradients are zeros."""
    lengths = [0, 1, min(nk, 64), nk // 2 + 1, nk, nk + 7, -3]
    b = len(lengths)
    q, k, v, go = _inputs(b, 4, 2, nq, nk, 64, dtype)
    clean = [min(max(n, 0), nk) for n in lengths]
    for i, n in enumerate(clean):
        k[i, :, n:] = torch.nan if i % 2 else torch.inf
        v[i, :, n:] = -torch.inf if i % 2 else torch.nan
    o, (dq, dk, dv) = _check(cuda_device, q, k, v, go, lengths, p, lengths_dtype=torch.int64 if p else torch.int32)
    assert bool((o[0] == 0).all()) and bool((dq[0] == 0).all())
    for i, n in enumerate(clean):
        assert bool((dk[i, :, n:] == 0).all()) and bool((dv[i, :, n:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nk", [(0, 5), (5, 0), (0, 0)])
def test_empty_sides(cuda_device, nq, nk):
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v, go = _inputs(2, 4, 2, nq, nk, 64, dtype)
        leaves = [t.to(cuda_device).requires_grad_() for t in (q, k, v)]
        o = cross_attention(*leaves, dropout_p=0.1, key=_key(cuda_device))
        assert o.shape == q.shape and bool((o == 0).all())
        for g, t in zip(torch.autograd.grad(o, leaves, go.to(cuda_device)), leaves):
            assert g.shape == t.shape and bool((g == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("p,scale", [(1.0, None), (1.0 / 65536, 0.3), (0.1, -0.2), (0.0, 0.0), (0.1, 3.0)])
def test_extreme_probabilities_and_scales(cuda_device, p, scale):
    _check(cuda_device, *_inputs(1, 2, 2, 70, 150, 64, torch.bfloat16), p=p, scale=scale)


@pytest.mark.gpu
def test_large_scores_do_not_overflow(cuda_device):
    """Scores of thousands: the softmax is one-hot and stays finite."""
    q, k, v, go = _inputs(1, 2, 2, 40, 90, 64, torch.bfloat16)
    _check(cuda_device, q * 30, k * 30, v, go)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq", [1, 70])
def test_leading_scores_of_minus_infinity_weigh_nothing(cuda_device, dtype, nq):
    """Keys of the type's lowest value whose scores overflow to -infinity, whole tiles of them before ordinary ones:
    their weights are zero, so values and gradients are those of the ordinary keys alone (zero terms leave every sum
    as it is, and 0 times the finite key is 0)."""
    low, n, d = 200, 260, 64
    q, k, v, go = _inputs(2, 2, 2, nq, n, d, dtype)
    q = q.abs() + 0.5  # every score of a low key is at most -0.5 * 3.38e38 * 64, below the lowest fp32
    k[:, :, :low] = torch.finfo(dtype).min
    leaves = [t.to(cuda_device).requires_grad_() for t in (q, k, v)]
    o = cross_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(o, leaves, go.to(cuda_device))
    assert not dk[:, :, :low].any() and not dv[:, :, :low].any()
    rest = [t.double() for t in (q, k[:, :, low:], v[:, :, low:], go)]
    exact = (ref.attention(*rest[:3], None, None, None), *ref.attention_grads(*rest, None, None, None))
    bounds = ref.attention_bounds(*rest, None, None, None, dtype)
    for got, e, bound, what in zip((o, dq, dk[:, :, low:], dv[:, :, low:]), exact, bounds, ("o", "dq", "dk", "dv")):
        _within(got, e, bound, what)


# one key range per row tile, several that a second kernel joins, packed heads, a wide head, the row form
INFINITE = [(2, 8, 2, 70, 130, 64, torch.bfloat16, False), (1, 2, 2, 3, 3000, 64, torch.bfloat16, True),
            (2, 4, 1, 5, 2500, 128, torch.bfloat16, True), (2, 2, 1, 40, 70, 64, torch.float32, False),
            (1, 2, 2, 5, 33, 136, torch.bfloat16, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("b,hq,hk,nq,nk,d,dtype,split", INFINITE)
def test_rows_of_scores_of_minus_infinity_are_zeros(cuda_device, b, hq, hk, nq, nk, d, dtype, split, p):
    """Even queries meet keys of the type's lowest value in scores that overflow to -infinity (at most -0.5 * 3.38e38 *
    d): zeros, and no gradient.  Odd queries are zero vectors, whose scores are zeros: with every value 1 they are means
    of ones, and with dropout sums of the kept ones' scale over the row's count."""
    assert _splits(b, hq, hk, nq, nk, d, dtype) == split
    q, k, _, go = _inputs(b, hq, hk, nq, nk, d, dtype)
    q = q.abs() + 0.5
    q[:, :, 1::2] = 0
    k = torch.full_like(k, torch.finfo(dtype).min)
    leaves = [t.to(cuda_device).requires_grad_() for t in (q, k, torch.ones_like(k))]
    key = _key(cuda_device) if p > 0 else None
    o = cross_attention(*leaves, dropout_p=p, key=key, site=SITE)
    only_even = go.clone()
    only_even[:, :, 1::2] = 0
    for grad in torch.autograd.grad(o, leaves, only_even.to(cuda_device), retain_graph=True):
        assert not bool(grad.any())
    _, _, dv = torch.autograd.grad(o, leaves, go.to(cuda_device))
    o = o.detach().double().cpu()
    assert not bool(o[:, :, 0::2].any())
    mult = _mult(q, k, p)
    weight = torch.ones(b, hq, nq, nk, dtype=torch.float64) if mult is None else mult
    # sums of nk terms in fp32, a tile's at a time: 2^-24 nk of the sum bounds any order; one rounding to dtype
    u = torch.finfo(dtype).eps / 2 + nk * 2.0**-24
    exact = weight.mean(-1)[:, :, 1::2, None].expand_as(o[:, :, 1::2])
    assert bool(((o[:, :, 1::2] - exact).abs() <= 2 * u * exact).all())  # 1/nk and its sum are rounded as well
    odd = (weight / nk)[:, :, 1::2].transpose(-1, -2) @ go.double()[:, :, 1::2]
    size = (weight / nk)[:, :, 1::2].transpose(-1, -2) @ go.double()[:, :, 1::2].abs()
    odd, size = (t.reshape(b, hk, hq // hk, nk, d).sum(2) for t in (odd, size))
    bound = 2 * (u + nq * (hq // hk) * 2.0**-24) * size + torch.finfo(dtype).tiny
    assert bool(((dv.double().cpu() - odd).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("b,hq,hk,nq,nk,d,dtype,split", INFINITE)
def test_nan_beside_scores_of_minus_infinity_stays_nan(cuda_device, b, hq, hk, nq, nk, d, dtype, split, p):
    """One live key of NaN among keys whose scores are -infinity: rows and gradients of the queries are NaN, whichever
    form and range it falls to."""
    q, k, v, go = _inputs(b, hq, hk, nq, nk, d, dtype)
    q, k = q.abs() + 0.5, torch.full_like(k, torch.finfo(dtype).min)
    k[:, :, nk * 2 // 3] = torch.nan
    leaves = [t.to(cuda_device).requires_grad_() for t in (q, k, v)]
    key = _key(cuda_device) if p > 0 else None
    o = cross_attention(*leaves, dropout_p=p, key=key, site=SITE)
    dq, _, _ = torch.autograd.grad(o, leaves, go.to(cuda_device))
    assert bool(torch.isnan(o).any(dim=-1).all()) and bool(torch.isnan(dq).any(dim=-1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,p", [(torch.float16, 0.0), (torch.bfloat16, 0.0), (torch.bfloat16, 0.1),
                                     (torch.float32, 0.0)])
def test_nan_in_a_live_key_reaches_every_row(cuda_device, dtype, p):
    """One key of each batch item is NaN, at every place of a tile's 32 columns: no row may come out finite."""
    places, n = 33, 130
    q, k, v, _ = _inputs(places, 2, 1, 3, n, 64, dtype)
    for i in range(places):
        k[i, :, i + (96 if i % 2 else 0)] = float("nan")
    key = _key(cuda_device) if p > 0 else None
    o = cross_attention(*(t.to(cuda_device) for t in (q, k, v)), dropout_p=p, key=key, site=SITE)
    assert bool(torch.isnan(o).any(dim=-1).all())


@pytest.mark.gpu
def test_layouts(cuda_device):
    """[b, h, n, d] planes, packed projections, transposed heads, odd offsets and broadcasts give what copies give."""
    b, h, n, d = 2, 4, 75, 64
    torch.manual_seed(5)
    packed = torch.randn(b, n, 3, h, d, device=cuda_device, dtype=torch.bfloat16)
    views = {
        "packed": [packed[:, :, i].transpose(1, 2) for i in range(3)],
        "bhnd": [torch.randn(b, h, n, d, device=cuda_device, dtype=torch.bfloat16) for _ in range(3)],
        "offset": [torch.randn(b, h, n, d + 1, device=cuda_device, dtype=torch.bfloat16)[..., 1:] for _ in range(3)],
        "head_dim_first": [torch.randn(b, h, d, n, device=cuda_device, dtype=torch.bfloat16).transpose(-1, -2)
                           for _ in range(3)],
        "every_second": [torch.randn(b, h, 2 * n, d, device=cuda_device, dtype=torch.bfloat16)[:, :, ::2]
                         for _ in range(3)],
        "broadcast": [torch.randn(b, h, n, d, device=cuda_device, dtype=torch.bfloat16)]
        + [torch.randn(1, 1, n, d, device=cuda_device, dtype=torch.bfloat16).expand(b, h, n, d) for _ in range(2)],
    }
    key = _key(cuda_device)
    go = torch.randn(b, h, n, d, device=cuda_device, dtype=torch.bfloat16)
    for name, qkv in views.items():
        leaves = [t.detach().requires_grad_() for t in qkv]
        copies = [t.detach().contiguous().requires_grad_() for t in qkv]
        o, oc = (cross_attention(*t, dropout_p=0.2, key=key, site=1) for t in (leaves, copies))
        assert torch.equal(o, oc), name
        grad = go if name != "bhnd" else go.expand(b, h, n, d)
        for x, y in zip(torch.autograd.grad(o, leaves, grad), torch.autograd.grad(oc, copies, grad)):
            assert torch.equal(x, y), name
    o = cross_attention(*leaves, dropout_p=0.2, key=key, site=1)
    one = torch.ones((), device=cuda_device, dtype=torch.bfloat16)
    g1 = torch.autograd.grad(o, leaves, one.expand_as(o), retain_graph=True)
    g2 = torch.autograd.grad(o, leaves, torch.ones_like(o))
    assert all(torch.equal(x, y) for x, y in zip(g1, g2))


@pytest.mark.gpu
def test_broadcast_context_gradient_is_the_sum_over_the_batch(cuda_device):
    """One context for every batch item: autograd sums the per-item gradients the formula gives."""
    q, k, v, go = _inputs(3, 2, 2, 20, 50, 64, torch.float32)
    k, v = k[:1], v[:1]
    kd, vd = (t.to(cuda_device).requires_grad_() for t in (k, v))
    o = cross_attention(q.to(cuda_device), kd.expand(3, -1, -1, -1), vd.expand(3, -1, -1, -1))
    gk, gv = torch.autograd.grad(o, (kd, vd), go.to(cuda_device))
    args = [t.double() for t in (q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1), go)]
    _, ek, ev = ref.attention_grads(*args)
    _, _, bk, bv = ref.attention_bounds(*args, None, None, None, torch.float32)
    for got, e, bound in ((gk, ek, bk), (gv, ev, bv)):
        _within(got, e.sum(0, keepdim=True), bound.sum(0, keepdim=True) + 2.0**-22 * e.abs().sum(0, keepdim=True), "sum")


@pytest.mark.gpu
def test_gradient_against_differences(cuda_device):
    """Central differences of the fp32 kernel along random directions.  f sums about 10^3 products of order one, so its
    fp32 rounding is below 2^-24 x 64 x 30 = 1.2e-4; over 2h = 0.1 that is 2.3e-3.  The third derivative along a unit
    direction is of order 1: h^2 / 6 = 4e-4.  Together below 5e-3."""
    q, k, v, go = (t.to(cuda_device) for t in _inputs(1, 2, 1, 6, 20, 16, torch.float32))
    key, h = _key(cuda_device), 0.05
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]

    def f(a, b, c):
        with torch.no_grad():
            o = cross_attention(a, b, c, dropout_p=0.3, key=key, site=2)
        return float((o.double() * go.double()).sum())

    o = cross_attention(*leaves, dropout_p=0.3, key=key, site=2)
    grads = torch.autograd.grad(o, leaves, go)
    for i in range(3):
        direction = torch.randn_like(leaves[i])
        direction /= direction.norm()
        up, down = ([t + s * h * direction if j == i else t for j, t in enumerate((q, k, v))] for s in (1, -1))
        numeric = (f(*up) - f(*down)) / (2 * h)
        assert abs(numeric - float((grads[i].double() * direction.double()).sum())) < 5e-3


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda_device):
    """Keys 2^20 elements apart: the last ones lie behind 2^31 elements of the cache."""
    nk, d, pitch = 2500, 64, 1 << 20
    cache = torch.empty(nk * pitch, dtype=torch.bfloat16, device=cuda_device)
    k, v = (cache.as_strided((1, 1, nk, d), (nk * pitch, pitch, pitch, 1), off) for off in (0, 128))
    k.normal_()
    v.normal_()
    q = torch.randn(1, 2, 3, d, device=cuda_device, dtype=torch.bfloat16)
    assert torch.equal(cross_attention(q, k, v), cross_attention(q, k.contiguous(), v.contiguous()))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    copies = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
    go = torch.randn_like(q)
    for x, y in zip(torch.autograd.grad(cross_attention(*leaves), leaves, go),
                    torch.autograd.grad(cross_attention(*copies), copies, go)):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_two_streams_at_once(cuda_device):
    """Calls on two streams share nothing: each gives what it gives alone."""
    sets = [[t.to(cuda_device).requires_grad_() for t in _inputs(4, 8, 2, 1 + 199 * i, 3000, 64, torch.bfloat16, i)[:3]]
            for i in range(2)]
    key = _key(cuda_device)

    def both(qkv):
        o = cross_attention(*qkv, dropout_p=0.1, key=key)
        return [o.detach(), *torch.autograd.grad(o, qkv, torch.ones_like(o))]

    alone = [both(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got[i] = both(sets[i])
    torch.cuda.synchronize()
    for a, g in zip(alone, got):
        assert all(torch.equal(x, y) for x, y in zip(a, g))


@pytest.mark.gpu
def test_captured_forward_and_backward_replay(cuda_device):
    """A captured pass reads its inputs, lengths and key anew at every replay."""
    b, nq, nk = 3, 20, 333
    q, k, v, go = _inputs(b, 4, 2, nq, nk, 64, torch.float16)
    leaves = [t.to(cuda_device).requires_grad_() for t in (q, k, v)]
    god, key = go.to(cuda_device), _key(cuda_device)
    lengths = torch.tensor([nk, 5, 200], dtype=torch.int32, device=cuda_device)

    def step():
        o = cross_attention(*leaves, key_lengths=lengths, dropout_p=0.2, key=key, site=SITE)
        grads = torch.autograd.grad(o, leaves, god)
        return [o.detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for new in ([nk, 5, 200], [0, 300, 1]):
        with torch.no_grad():
            lengths.copy_(torch.tensor(new, dtype=torch.int32))
            for t in leaves:
                t.copy_(torch.randn_like(t))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in out]
        assert all(torch.equal(x, y) for x, y in zip(replayed, step()))


def _bounds_with_exact_row_sums(q, k, v, go, lengths, mult, dtype):
    """Bounds of dq and dk where D = rowsum(P dP) comes from the unrounded probabilities, term by term as in
    attention_bounds, with e_dP = 2 (d + 16) 2^-24 |dO| |V|^T mult (d fp32 products and sums, truncated ones too):
      D:  P (e_dP + (e_p + nk 2^-24) |dP|), summed;
      dS: (u + e_p) |dS| + P (error of D + e_dP + 2^-22 (|dP| + |D|)) + tiny."""
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * u
    b, hq, nq, d = q.shape
    hk, nk = k.shape[1], k.shape[2]
    scale = d**-0.5
    p, live = ref.probabilities(q, k, lengths, scale)
    zero = torch.zeros((), dtype=q.dtype)
    kr, vr = (torch.where(live.transpose(-1, -2), t.repeat_interleave(hq // hk, dim=1), zero) for t in (k, v))
    mult = torch.ones((), dtype=q.dtype) if mult is None else mult
    ep = 2 * ((d + 16) * 2.0**-24 * scale * (q.abs() @ kr.abs().transpose(-1, -2))).amax(-1, keepdim=True) + 2.0**-19
    e_dp = 2 * (d + 16) * 2.0**-24 * (go.abs() @ vr.abs().transpose(-1, -2)) * mult
    dp = (go @ vr.transpose(-1, -2)) * mult
    row = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - row)
    e_d = (p * (e_dp + (ep + nk * 2.0**-24) * dp.abs())).sum(-1, keepdim=True)
    e_ds = (u + ep) * ds.abs() + p * (e_d + e_dp + 2.0**-22 * (dp.abs() + row.abs())) + tiny * live
    dq, dk, _ = ref.attention_grads(q, k, v, go, lengths, None, mult)
    e_dk = (e_ds.transpose(-1, -2) @ q.abs()).reshape(b, hk, hq // hk, nk, d).sum(2)
    return tuple(u * g.abs() + tiny + scale * e * (1 + 2.0**-10) for g, e in ((dq, e_ds @ kr.abs()), (dk, e_dk)))


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 33),
                                     (torch.float16, 200), (torch.float32, 48)])
@pytest.mark.parametrize("nk,lengths", [(1, None), (2, None), (5, None), (17, [17, 1, 0]), (32, [2, 32, 31])])
def test_few_keys_keep_the_rounding_of_the_output_out_of_their_gradients(cuda_device, nk, lengths, dtype, d, p):
    """dS = P (dP - D) cancels, most of all where few keys share a row's weight (one key: dS = 0); D from the rounded
    output would leave 2^-9 |dO| |O| of bf16 there.  The tensor-core form's border of 64 keys is the next test's."""
    b = 3
    q, k, v, go = _inputs(b, 4, 2, 37, nk, d, dtype)
    leaves = [t.to(cuda_device).requires_grad_() for t in (q, k, v)]
    dev_len = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    key = _key(cuda_device) if p > 0 else None
    o = cross_attention(*leaves, key_lengths=dev_len, dropout_p=p, key=key, site=SITE)
    dq, dk, _ = torch.autograd.grad(o, leaves, go.to(cuda_device))
    wide = [t.double() for t in (q, k, v, go)]
    mult = _mult(q, k, p)
    eq, ek, _ = ref.attention_grads(*wide, lengths, None, mult)
    bq, bk = _bounds_with_exact_row_sums(*wide, lengths, mult, dtype)
    _within(dq, eq, bq, "dq")
    _within(dk, ek, bk, "dk")


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float16, 72), (torch.bfloat16, 136), (torch.float32, 64)])
@pytest.mark.parametrize("nk", [31, 32, 33, 48, 63, 64, 65])
def test_borders_of_the_forms_for_few_keys(cuda_device, nk, dtype, d, p):
    """Every length behind the borders at a tile of the row form and a chunk of the tensor-core form, several query
    tiles, packed heads, ragged batches."""
    q, k, v, go = _inputs(5, 4, 2, 150, nk, d, dtype)
    _check(cuda_device, q, k, v, go, [nk, 0, 1, nk - 1, nk // 2], p)
    if dtype != torch.float32 and d <= 128 and nk <= 64:
        test_few_keys_keep_the_rounding_of_the_output_out_of_their_gradients(cuda_device, nk, [nk, 3, nk - 1], dtype, d, p)
