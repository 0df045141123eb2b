"""64-bit definitions of the counter-based dropout, cross attention and several-axes rotary operators, on the CPU.

Random bits with numpy's 64-bit integers, everything else in torch float64; written from the formulas, without the
package."""
from __future__ import annotations

import numpy as np
import torch

_W = np.uint64(0xFFFFFFFF)


def philox16(c0, c1, c2, seed: int, step: int, site: int) -> np.ndarray:
    """[..., 8] 16-bit numbers: Philox4x32 with seven rounds, counter (c0, c1, c2, step), key (seed, site)."""
    c0, c1, c2 = np.broadcast_arrays(*(np.asarray(c, dtype=np.uint64) for c in (c0, c1, c2)))
    c3 = np.full(c0.shape, step & 0xFFFFFFFF, dtype=np.uint64)
    k0, k1 = seed & 0xFFFFFFFF, ((seed >> 32) & 0xFFFFFFFF) ^ site
    for _ in range(7):
        a, b = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        hi_a, hi_b = a >> np.uint64(32), b >> np.uint64(32)
        c0, c1, c2, c3 = hi_b ^ c1 ^ np.uint64(k0), b & _W, hi_a ^ c3 ^ np.uint64(k1), a & _W
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    halves = []
    for w in (c0, c1, c2, c3):
        halves += [w & np.uint64(0xFFFF), w >> np.uint64(16)]
    return np.stack(halves, axis=-1).astype(np.int64)


def drop_scale(p: float) -> tuple[int, float]:
    t = int(round(p * 65536))
    return t, (65536.0 / (65536 - t) if t < 65536 else 0.0)


def dropout_mult(n: int, p: float, seed: int, step: int, site: int) -> torch.Tensor:
    """float64 [n]: 0 for dropped elements, the scale for kept ones."""
    t, c = drop_scale(p)
    g = np.arange((n + 7) // 8, dtype=np.uint64)
    u = philox16(g & _W, g >> np.uint64(32), 0xFFFFFFFF, seed, step, site).reshape(-1)[:n]
    return torch.from_numpy((u >= t).astype(np.float64) * c)


def attention_mult(b: int, heads: int, nq: int, nk: int, p: float, seed: int, step: int, site: int) -> torch.Tensor:
    """float64 [b, heads, nq, nk]: the dropout multiplier of every probability."""
    t, c = drop_scale(p)
    u = philox16(np.arange((nk + 7) // 8)[None, None], np.arange(nq)[None, :, None],
                 np.arange(b * heads)[:, None, None], seed, step, site)
    u = u.reshape(b, heads, nq, -1)[..., :nk]
    return torch.from_numpy((u >= t).astype(np.float64) * c)


def probabilities(q, k, lengths, scale):
    """softmax over each item's keys, rows without keys all zero; q [b, h, nq, d], k [b, hk, nk, d] float64."""
    b, hq, nq, d = q.shape
    nk = k.shape[2]
    k = k.repeat_interleave(hq // k.shape[1], dim=1)
    live = torch.ones(b, nk, dtype=torch.bool)
    if lengths is not None:
        live = torch.arange(nk)[None] < torch.as_tensor(lengths).long()[:, None]
    live = live[:, None, None]
    # masked keys leave the product before it is formed: whatever they hold cannot reach a result
    k = torch.where(live.transpose(-1, -2), k, torch.zeros((), dtype=k.dtype))
    s = (q @ k.transpose(-1, -2)) * scale
    s = s.masked_fill(~live, -torch.inf)
    m = s.detach().amax(dim=-1, keepdim=True) if nk else s.new_zeros(b, hq, nq, 1)
    e = torch.where(live, torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m))), torch.zeros_like(s))
    total = e.sum(dim=-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total), live


def attention(q, k, v, lengths=None, scale=None, mult=None):
    """float64 (mult * softmax(scale q k^T)) v; differentiable."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    p, live = probabilities(q, k, lengths, scale)
    v = v.repeat_interleave(q.shape[1] // v.shape[1], dim=1)
    v = torch.where(live.transpose(-1, -2), v, torch.zeros((), dtype=v.dtype))
    return (p if mult is None else p * mult) @ v


def attention_grads(q, k, v, grad, lengths=None, scale=None, mult=None):
    """The gradients by formula: dV = Pd^T dO, dS = P (dP - rowsum(P dP)), dQ = scale dS K, dK = scale dS^T Q, the
    last two and dV summed over the query heads that share a key / value head."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    p, live = probabilities(q, k, lengths, scale)
    b, hq, nq, d = q.shape
    hk, nk = k.shape[1], k.shape[2]
    zero = torch.zeros((), dtype=q.dtype)
    kr, vr = (torch.where(live.transpose(-1, -2), t.repeat_interleave(hq // hk, dim=1), zero) for t in (k, v))
    mult = torch.ones((), dtype=q.dtype) if mult is None else mult
    dp = (grad @ vr.transpose(-1, -2)) * mult
    ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True))
    dq = scale * ds @ kr
    dk = scale * ds.transpose(-1, -2) @ q
    dv = (p * mult).transpose(-1, -2) @ grad
    return dq, dk.reshape(b, hk, hq // hk, nk, d).sum(2), dv.reshape(b, hk, hq // hk, nk, d).sum(2)


def attention_bounds(q, k, v, grad, lengths, scale, mult, dtype):
    """Elementwise error bounds (o, dq, dk, dv) of a computation with fp32 sums whose probabilities and dS are rounded
    to ``dtype`` before their products and whose results are rounded to it.

    u: one rounding to dtype (relative), tiny: its absolute part below the smallest normal number (probabilities are
    rounded before the division by the row sum, which is at least 1).  A score is off by e_s = (d + 16) 2^-24 scale
    |q| |k| (d fp32 products and sums), so a probability by the relative e_p = 2 max(e_s) + 2^-19 (its own score, the
    row sum's, the exponential and up to 2^14 additions at 2^-24 each, halved by their tree).  Then
      o:  u |o| + (u + e_p) Pd |v|                                     (P rounded)
      D:  |dO| (error of o);   dP: e_p |dO| |v|^T mult
      dS: u |dS| + e_p |dS| + P (error of D + error of dP) + tiny
      dq: u |dq| + scale |error of dS| |k|, dk alike, dv: u |dv| + (u + e_p) Pd^T |dO|."""
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * u
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    p, live = probabilities(q, k, lengths, scale)
    b, hq, nq, d = q.shape
    hk, nk = k.shape[1], k.shape[2]
    zero = torch.zeros((), dtype=q.dtype)
    kr, vr = (torch.where(live.transpose(-1, -2), t.repeat_interleave(hq // hk, dim=1), zero).abs() for t in (k, v))
    signed_v = torch.where(live.transpose(-1, -2), v.repeat_interleave(hq // hk, dim=1), zero)
    mult = torch.ones((), dtype=q.dtype) if mult is None else mult
    size = abs(scale)  # bounds are magnitudes, whatever the scale's sign
    es = (d + 16) * 2.0**-24 * size * (q.abs() @ kr.transpose(-1, -2))
    ep = 2 * es.amax(dim=-1, keepdim=True) + 2.0**-19 if nk else es.new_zeros(b, hq, nq, 1)
    pd = p * mult
    o = pd @ signed_v
    eo = u * o.abs() + tiny + (u + ep) * (pd @ vr) + tiny * ((live * mult).expand_as(p) @ vr)
    if grad is None:
        return eo, None, None, None
    dp = (grad @ signed_v.transpose(-1, -2)) * mult
    dsum = (p * dp).sum(dim=-1, keepdim=True)
    ds = p * (dp - dsum)
    e_d = (grad.abs() * eo).sum(dim=-1, keepdim=True) + 2.0**-20 * (grad.abs() * o.abs()).sum(dim=-1, keepdim=True)
    e_ds = (u + ep) * ds.abs() + p * (e_d + ep * (grad.abs() @ vr.transpose(-1, -2)) * mult) + tiny * live
    dq = scale * ds @ torch.where(live.transpose(-1, -2), k.repeat_interleave(hq // hk, dim=1), zero)
    edq = u * dq.abs() + tiny + size * (e_ds @ kr) * (1 + 2.0**-10)

    def shared(t):
        return t.reshape(b, hk, hq // hk, nk, d).sum(2)

    dk = shared(scale * ds.transpose(-1, -2) @ q)
    dv = shared(pd.transpose(-1, -2) @ grad)
    # the row's relative error moves with the query: inside the products
    edk = u * dk.abs() + tiny + shared(size * e_ds.transpose(-1, -2) @ q.abs()) * (1 + 2.0**-10)
    edv = u * dv.abs() + tiny + shared((pd * (u + ep) + tiny * live * mult).transpose(-1, -2) @ grad.abs()) * \
        (1 + 2.0**-10)
    return eo, edq, edk, edv


def rotary_axes(t, positions, freqs, sections, inverse=False):
    """float64 rotation of t [b, h, n, d]; positions [b, n, axes] or [n, axes]."""
    t = t.double()
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    angle = positions.double()[..., axis] * freqs.double()
    angle = angle if angle.dim() == 3 else angle[None]
    angle = (-angle if inverse else angle)[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    n = 2 * angle.shape[-1]
    e, o = t[..., 0:n:2], t[..., 1:n:2]
    y = t.clone()
    y[..., 0:n:2] = e * cos - o * sin
    y[..., 1:n:2] = o * cos + e * sin
    return y
