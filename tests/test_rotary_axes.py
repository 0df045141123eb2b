"""Rotary positions with several axes against the 64-bit definition, and their refusals."""
from __future__ import annotations

import pytest
import torch

from oracle import context_ref as ref
from pymsst_b200 import _native as nat
from pymsst_b200.cross_attention import rotary_axes

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _freqs(sections):
    return torch.cat([10000.0 ** (-torch.arange(s, dtype=torch.float32) / s) for s in sections])


def _positions(b, n, axes, far, dtype, g):
    pos = torch.randint(-5, 70, (b, n, axes), generator=g)
    pos[..., 0] += far
    if dtype == torch.float32:
        return pos.float() + 0.25
    return pos.to(dtype)


def _close(got, exact, t, dtype):
    """One rounding to dtype; cosine and sine to 2^-22 (an angle reduced in fp64, 2^-23 of a half turn, and their own
    two units), the two products and the sum 2^-23 more, of both elements' magnitude."""
    u = torch.finfo(dtype).eps / 2
    pair = t.double().abs().reshape(*t.shape[:-1], -1, 2).sum(-1, keepdim=True).expand(*t.shape[:-1], -1, 2)
    bound = u * exact.abs() + torch.finfo(dtype).smallest_normal * u + 2.0**-21 * pair.reshape(t.shape)
    err = (got.double().cpu() - exact).abs()
    assert bool((err <= bound).all()), f"off by {float((err / bound).max()):.3f} of the bound"


def test_definition_turns_pairs_by_their_axis():
    t = torch.randn(1, 1, 3, 8, dtype=torch.float64)
    pos = torch.tensor([[1, 0], [0, 2], [3, 4]])
    y = ref.rotary_axes(t, pos, torch.tensor([0.5, 0.25, 2.0]), [2, 1])
    assert torch.equal(y[..., 6:], t[..., 6:])
    z = torch.view_as_complex(t[..., :6].reshape(1, 1, 3, 3, 2))
    angle = torch.stack([pos[:, 0] * 0.5, pos[:, 0] * 0.25, pos[:, 1] * 2.0], dim=-1).double()
    expect = torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)).reshape(1, 1, 3, 6)
    assert torch.allclose(y[..., :6], expect, rtol=0, atol=1e-14)
    assert torch.allclose(ref.rotary_axes(y, pos, torch.tensor([0.5, 0.25, 2.0]), [2, 1], inverse=True), t, atol=1e-14)


def test_refusals():
    t, pos, f = torch.randn(2, 3, 4, 8), torch.zeros(2, 4, 2, dtype=torch.int32), torch.ones(4)
    with pytest.raises(nat.FusedKernelUnavailable):
        rotary_axes(t, pos, f, [2, 2])
    for args in ((t[0], pos, f, [2, 2]), (t[..., :7], pos, f, [2, 2]), (t, pos, f, [2, 3]), (t, pos, f, [4]),
                 (t, pos.half(), f, [2, 2]), (t, pos, f.double(), [2, 2]), (t, pos, f[:3], [2, 2]), (t, pos, f, []),
                 (t, pos, f, [0, 4]), (t, pos[:, :3], f, [2, 2]), (t, pos, f.clone().requires_grad_(), [2, 2])):
        with pytest.raises(ValueError):
            rotary_axes(*args)
    with pytest.raises(TypeError):
        rotary_axes(t.double(), pos, f, [2, 2])
    lib = nat.library()

    def call(dim=8, axes=2, sections=(2, 2), pos_type=0, strides=(96, 24, 8) * 2, dtype=0, x=16):
        return lib.pmb_rotary_axes(x, 16, 16, 16, 2, 4, 3, dim, nat.i64_array(strides), 0, pos_type, axes,
                                   nat.i64_array(sections), 0, dtype, None)

    assert call(dim=7) == -1 and b"even" in lib.pmb_last_error()
    assert call(axes=0) == -1 and call(axes=5, sections=(1,) * 5) == -1
    assert call(sections=(2, 3)) == -1 and b"sections hold" in lib.pmb_last_error()
    assert call(sections=(0, 2)) == -1
    assert call(strides=(96, 24, 7, 96, 24, 8)) == -1
    assert call(x=4) == -1 and b"aligned" in lib.pmb_last_error()
    assert call(pos_type=3) == -2 and call(dtype=5) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,h,n,d,sections,far,pos_dtype", [
    (1, 1, 1, 2, [1], 0, torch.int32),
    (2, 3, 5, 10, [2, 1], 0, torch.int64),
    (1, 16, 62, 64, [16, 16], 1 << 20, torch.int32),
    (3, 5, 129, 80, [9, 20], 1 << 24, torch.int32),
    (2, 8, 300, 64, [12, 12, 8], 1 << 28, torch.int64),
    (2, 2, 33, 128, [16, 16, 16, 16], 100_000, torch.float32),
    (1, 70, 9, 256, [100, 28], 0, torch.int32),
    (5, 1, 1, 64, [32], 12345, torch.int32),
    (1, 1, 2000, 8, [4], 0, torch.int32),
])
def test_rotation_and_its_gradient(cuda_device, dtype, b, h, n, d, sections, far, pos_dtype):
    g = torch.Generator().manual_seed(n)
    t, gy = (torch.randn(b, n, h, d, generator=g).to(dtype).transpose(1, 2) for _ in range(2))
    pos, freqs = _positions(b, n, len(sections), far, pos_dtype, g), _freqs(sections)
    td = t.to(cuda_device).requires_grad_()
    y = rotary_axes(td, pos.to(cuda_device), freqs.to(cuda_device), sections)
    assert y.shape == t.shape and y.dtype == dtype
    _close(y.detach(), ref.rotary_axes(t, pos, freqs, sections), t, dtype)
    (gt,) = torch.autograd.grad(y, td, gy.to(cuda_device))
    _close(gt, ref.rotary_axes(gy, pos, freqs, sections, inverse=True), gy, dtype)


@pytest.mark.gpu
def test_views_shared_positions_and_infinities(cuda_device):
    g = torch.Generator().manual_seed(3)
    n, d = 37, 16
    freqs = _freqs([4, 2]).to(cuda_device)
    pos = torch.randint(0, 100, (n, 2), generator=g).to(cuda_device)
    packed = torch.randn(2, n, 3, 4, d, device=cuda_device, dtype=torch.bfloat16)  # projection of q, k, v
    q = packed[:, :, 0].transpose(1, 2)
    expect = rotary_axes(q.clone(memory_format=torch.contiguous_format), pos, freqs, [4, 2])
    both = rotary_axes(packed[:, :, :2].flatten(2, 3).transpose(1, 2), pos[None].expand(2, n, 2), freqs, [4, 2])
    assert torch.equal(rotary_axes(q, pos, freqs, [4, 2]), expect)
    assert torch.equal(both[:, :4], expect)
    odd = torch.randn(2, 4, n, d + 1, device=cuda_device)[..., 1:]
    assert torch.equal(rotary_axes(odd, pos, freqs, [4, 2]), rotary_axes(odd.clone(), pos, freqs, [4, 2]))
    last = torch.randn(2, 4, d, n, device=cuda_device).transpose(-1, -2)
    assert torch.equal(rotary_axes(last, pos, freqs, [4, 2]), rotary_axes(last.contiguous(), pos, freqs, [4, 2]))
    one = torch.randn(1, 4, n, d, device=cuda_device).expand(3, 4, n, d).requires_grad_(False)
    assert torch.equal(rotary_axes(one, pos, freqs, [4, 2])[2], rotary_axes(one[:1], pos, freqs, [4, 2])[0])
    # unrotated pairs pass through whatever they hold
    x = torch.randn(1, 2, n, d, device=cuda_device)
    x[..., 12:] = torch.inf
    assert bool((rotary_axes(x, pos, freqs, [4, 2])[..., 12:] == torch.inf).all())
    empty = rotary_axes(x[:, :, :0], pos[:0], freqs, [4, 2])
    assert empty.shape == (1, 2, 0, d)


@pytest.mark.gpu
def test_one_axis_matches_the_packages_rotary(cuda_device):
    """With one axis over the whole head and positions 0 .. n - 1 this is ops.rotary's rotation: fp32 tables there,
    so off by the rounding of the tables' angles (up to 40 x 2^-24 rad) and a few units of the
    cosines and products, of both elements of a pair."""
    from pymsst_b200.extension import ops

    n, h, d = 40, 4, 32
    freqs = _freqs([d // 2]).to(cuda_device)
    t = torch.randn(2, n, h, d, device=cuda_device)
    angle = torch.arange(n, device=cuda_device, dtype=torch.float32)[:, None] * freqs
    angle = angle[None, :, None]
    expect = ops.rotary_forward(t, angle.cos(), angle.sin())
    got = rotary_axes(t.transpose(1, 2), torch.arange(n, device=cuda_device)[:, None], freqs, [d // 2]).transpose(1, 2)
    assert float((got - expect).abs().max()) <= (40 + 8) * 2.0**-24 * float(t.abs().max()) * 2
