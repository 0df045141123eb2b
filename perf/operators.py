"""Operators of the dropout / cross-attention / rotary set: the cases they are timed and compared on.

``run`` makes the calls a program makes of the package (``own`` true) or computes the same outputs with elementary
torch operations (``own`` false); ``exact`` computes them from the definitions in 64 bits.

Random bits.  Dropout takes 16 bits per element from Philox4x32 with seven rounds.  ``key`` holds (seed, step); the
generator's key is (seed's low word, seed's high word xor site).  Elementwise dropout numbers its elements row by row:
group ``index // 8`` has the counter (group's low word, group's high word, 2^32 - 1, step), attention's group of eight
keys (key // 8, query, batch index * heads + head, step).  Element e of a group takes word e // 2, the low half when e
is even.  An element is dropped when its 16 bits are below round(65536 p) and scaled by 65536 / (65536 - round(65536 p))
otherwise.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_MASK = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------------- cases
def _drop(name, rows, cols, dtype, p, residual, train, gelu=False):
    case = dict(kind="gelu_dropout" if gelu else "dropout", rows=rows, cols=cols, dtype=dtype, p=p,
                residual=residual, train=train)
    return dict(case, name=name) if name else case


def _attn(name, batch, heads, kv_heads, nq, nk, dim, dtype, p, ragged, train):
    case = dict(kind="attention", batch=batch, heads=heads, kv_heads=kv_heads, nq=nq, nk=nk, dim=dim, dtype=dtype, p=p,
                ragged=ragged, train=train)
    return dict(case, name=name) if name else case


def _rot(name, batch, tokens, heads, dim, sections, dtype, train):
    case = dict(kind="rotary", batch=batch, tokens=tokens, heads=heads, dim=dim, sections=sections, dtype=dtype,
                train=train)
    return dict(case, name=name) if name else case


def listed():
    return [
        # dropout and residual sum behind the output projection of one transformer layer: 4 chunks x 258 frames x
        # 62 bands of 192 features, forward and backward
        _drop("dropout_residual_train", 63984, 192, "bf16", 0.1, True, True),
        # one short clip of an odd length in full precision, no residual: latency counts
        _drop("dropout_small", 1037, 191, "fp32", 0.25, False, False),
        # the feed-forward's activation with its dropout, the widest activations of a layer, forward and backward
        _drop("gelu_dropout_train", 63984, 768, "bf16", 0.1, False, True, gelu=True),
        # the same on one clip of 87 frames, half precision
        _drop("gelu_dropout_clip", 87 * 62, 768, "fp16", 0.1, False, True, gelu=True),
        # time-axis attention of a training step with dropout on the probabilities (keys and queries of one length)
        _attn("attention_time_axis_train", 248, 8, 8, 258, 258, 64, "bf16", 0.1, False, True),
        # frames of a clip attending to a longer, padded context with shared key / value heads, training
        _attn("attention_context_train", 16, 8, 2, 258, 1531, 64, "bf16", 0.1, True, True),
        # long clip against a long context, inference
        _attn("attention_long", 2, 8, 8, 4096, 4096, 64, "fp16", 0.0, False, False),
        # one new frame per stream attending to a long padded context: the cache is what has to be read
        _attn("attention_single_token", 32, 8, 8, 1, 8192, 64, "bf16", 0.0, True, False),
        # the smallest call: one stream, a few queries, wide heads
        _attn("attention_small", 1, 8, 4, 5, 77, 128, "fp16", 0.0, False, False),
        # queries and keys of a (frame, band, channel) grid, forward and backward
        _rot("rotary_grid_train", 4, 15996, 16, 64, "12,12,8", "bf16", True),
        # one new frame's tokens far into a stream
        _rot("rotary_frame", 1, 62, 16, 64, "16,16", "bf16", False),
        # full precision, odd counts, a part of the head not rotated
        _rot("rotary_partial_fp32", 3, 2047, 5, 80, "9,20", "fp32", True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["dropout", "gelu_dropout", "attention", "attention", "rotary"])
    while True:
        train = rng.random() < 0.5
        if kind in ("dropout", "gelu_dropout"):
            gelu = kind == "gelu_dropout"
            case = _drop(None, _log_int(rng, 64, 70000), _log_int(rng, 32, 1536), rng.choice(["bf16", "fp16", "fp32"]),
                         rng.choice([0.05, 0.1, 0.25, 0.5]), not gelu and rng.random() < 0.5, train, gelu)
            if case["rows"] * case["cols"] * _SIZE[case["dtype"]] <= 63984 * 768 * 2:
                return case
        elif kind == "attention":
            heads, kv_heads = rng.choice([(8, 8), (8, 8), (8, 2), (8, 1), (4, 4), (6, 2), (12, 4)])
            case = _attn(None, _log_int(rng, 1, 256), heads, kv_heads, _log_int(rng, 1, 2048), _log_int(rng, 1, 8192),
                         rng.choice([64, 64, 64, 128, 32, 40]), rng.choice(["bf16", "fp16"]),
                         rng.choice([0.0, 0.1, 0.25]), rng.random() < 0.5, train)
            pairs = case["batch"] * heads * case["nq"] * case["nk"]
            cost = pairs * case["dim"] * (14 if train else 4)
            if cost <= 248 * 8 * 258 * 258 * 64 * 14 and work(case)["bytes"] <= work(listed()[4])["bytes"]:
                return case
        else:
            dim = rng.choice([32, 64, 64, 80, 128])
            axes = rng.choice([1, 2, 2, 3])
            cuts = [rng.randint(1, dim // 2 // axes) for _ in range(axes)]
            case = _rot(None, _log_int(rng, 1, 8), _log_int(rng, 1, 16000), rng.choice([1, 4, 5, 8, 16]), dim,
                        ",".join(map(str, cuts)), rng.choice(["bf16", "fp16", "fp32"]), train)
            n = case["batch"] * case["tokens"] * case["heads"] * dim * _SIZE[case["dtype"]]
            if n <= 4 * 15996 * 16 * 64 * 2:
                return case


def _lengths(case):
    """Key counts of a padded batch: from the full length down to about half of it; in a batch of eight or more one
    item has no context at all."""
    b, nk = case["batch"], case["nk"]
    if not case["ragged"]:
        return [nk] * b
    out = [max(1, nk - nk * i // (2 * b)) for i in range(b)]
    if b >= 8:
        out[-1] = 0
    return out


def work(case):
    es = _SIZE[case["dtype"]]
    if case["kind"] in ("dropout", "gelu_dropout"):
        n = case["rows"] * case["cols"]
        gelu = case["kind"] == "gelu_dropout"
        passes = 3 if case["residual"] else 2
        if case["train"]:
            passes += 3 if gelu else 2  # gradient (and the activation's input) read, input gradient written
        return {"bytes": passes * n * es, "flops": (10 if gelu else 2) * n * (2 if case["train"] else 1)}
    if case["kind"] == "attention":
        keys = sum(_lengths(case))
        q = case["batch"] * case["nq"] * case["heads"] * case["dim"]
        kv = keys * case["kv_heads"] * case["dim"]
        pairs = case["nq"] * case["heads"] * keys
        byt, flops = (2 * q + 2 * kv) * es, 4 * pairs * case["dim"]
        if case["train"]:  # q, k, v, o and the gradient of o read; three gradients written
            full = case["batch"] * case["nk"] * case["kv_heads"] * case["dim"]
            byt += (4 * q + 2 * kv + 2 * full) * es
            flops += 10 * pairs * case["dim"]
        return {"bytes": byt, "flops": flops}
    n = case["batch"] * case["tokens"] * case["heads"] * case["dim"]
    axes = len(case["sections"].split(","))
    times = 2 if case["train"] else 1
    return {"bytes": times * (2 * n * es + case["batch"] * case["tokens"] * axes * 4), "flops": times * 3 * n}


# --------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    kind = case["kind"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev).to(dt)

    state = {"case": case}
    if kind in ("dropout", "gelu_dropout", "attention"):
        # what a program's dropout generator hands out for one step: (seed, step)
        state["key"] = torch.randint(0, 2**31, (2,), generator=gen, device=dev, dtype=torch.int64)
        state["site"] = 3 + seed % 7
    if kind in ("dropout", "gelu_dropout"):
        state["x"] = randn(case["rows"], case["cols"]).requires_grad_(case["train"])
        if case["residual"]:
            state["residual"] = randn(case["rows"], case["cols"]).requires_grad_(case["train"])
        if case["train"]:
            state["grad"] = randn(case["rows"], case["cols"])
    elif kind == "attention":
        b, d = case["batch"], case["dim"]
        # projections write [batch, position, head, dim] planes; attention gets [batch, head, position, dim] views
        for name, n, h in (("q", case["nq"], case["heads"]), ("k", case["nk"], case["kv_heads"]),
                           ("v", case["nk"], case["kv_heads"])):
            state[name] = randn(b, n, h, d).transpose(1, 2).requires_grad_(case["train"])
        state["lengths"] = None
        if case["ragged"]:
            lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
            state["lengths"] = lengths[torch.randperm(b, generator=gen, device=dev)].contiguous()
        if case["train"]:
            state["grad"] = randn(b, case["nq"], case["heads"], d).transpose(1, 2)
    else:
        b, n = case["batch"], case["tokens"]
        sections = [int(s) for s in case["sections"].split(",")]
        state["sections"] = sections
        state["t"] = randn(b, n, case["heads"], case["dim"]).transpose(1, 2).requires_grad_(case["train"])
        # tokens of a grid, the first axis (frames) counted from far into a stream
        index = torch.arange(n, device=dev)
        start = torch.randint(0, 1 << 20, (b, 1), generator=gen, device=dev)
        cols = [start + index // 62, (index % 62).expand(b, n), (index % 2).expand(b, n)][: len(sections)]
        state["positions"] = torch.stack(cols, dim=-1).to(torch.int32).contiguous()
        state["freqs"] = torch.cat([10000.0 ** (-torch.arange(s, device=dev, dtype=torch.float32) / s)
                                    for s in sections])
        if case["train"]:
            state["grad"] = randn(b, n, case["heads"], case["dim"]).transpose(1, 2)
    return state


# ----------------------------------------------------------------------------------------------- plain forms
def _random16(c0, c1, c2, step, seed, site):
    """[..., 8] 16-bit numbers of the groups with counter words (c0, c1, c2, step), broadcast against each other."""
    c0, c1, c2 = torch.broadcast_tensors(c0, c1, c2)
    c3 = (step & _MASK).expand_as(c0)
    k0, k1 = seed & _MASK, ((seed >> 32) & _MASK) ^ site
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products, wrapped
        c0, c1, c2, c3 = ((b >> 32) & _MASK) ^ c1 ^ k0, b & _MASK, ((a >> 32) & _MASK) ^ c3 ^ k1, a & _MASK
        k0, k1 = (k0 + 0x9E3779B9) & _MASK, (k1 + 0xBB67AE85) & _MASK
    halves = [h for w in (c0, c1, c2, c3) for h in (w & 0xFFFF, w >> 16)]
    return torch.stack(halves, dim=-1)


def _threshold(p):
    t = int(round(p * 65536))
    return t, 65536.0 / (65536 - t)


def _keep_flat(state, n):
    key = state["key"]
    g = torch.arange((n + 7) // 8, device=key.device, dtype=torch.int64)
    u = _random16(g & _MASK, g >> 32, torch.full_like(g, _MASK), key[1], key[0], state["site"])
    return u.reshape(-1)[:n] >= _threshold(state["case"]["p"])[0]


def _plain_dropout(state):
    case = state["case"]
    scale = _threshold(case["p"])[1]
    x = state["x"]
    keep = _keep_flat(state, x.numel()).reshape(x.shape)
    zero = torch.zeros((), device=x.device)
    xf = x.float()
    gelu = case["kind"] == "gelu_dropout"
    cdf = 0.5 * (1.0 + torch.erf(xf * 0.7071067811865476)) if gelu else None
    y = torch.where(keep, (xf * cdf if gelu else xf) * scale, zero)
    if case["residual"]:
        y = y + state["residual"].float()
    outs = [y.to(x.dtype)]
    if case["train"]:
        g = state["grad"].float()
        if gelu:
            g = g * (cdf + xf * torch.exp(-0.5 * xf * xf) * 0.3989422804014327)
        outs.append(torch.where(keep, g * scale, zero).to(x.dtype))
        if case["residual"]:
            outs.append(state["grad"])
    return outs


def _plain_attention(state):
    case = state["case"]
    q, k, v = state["q"].float(), state["k"].float(), state["v"].float()
    b, hq, nq, d = q.shape
    hk, nk = k.shape[1], k.shape[2]
    k, v = k.repeat_interleave(hq // hk, dim=1), v.repeat_interleave(hq // hk, dim=1)
    scale = d ** -0.5
    s = (q @ k.transpose(-1, -2)) * scale
    live = torch.ones(b, 1, 1, nk, dtype=torch.bool, device=q.device)
    if state["lengths"] is not None:
        live = (torch.arange(nk, device=q.device)[None] < state["lengths"][:, None])[:, None, None]
    s = torch.where(live, s, torch.full((), -math.inf, device=q.device))
    m = s.amax(dim=-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    keep = None
    if case["p"] > 0:
        key = state["key"]
        dev = q.device
        threshold, c = _threshold(case["p"])
        u = _random16(torch.arange((nk + 7) // 8, device=dev)[None, None],
                      torch.arange(nq, device=dev)[None, :, None],
                      torch.arange(b * hq, device=dev)[:, None, None], key[1], key[0], state["site"])
        keep = (u.reshape(b, hq, nq, -1)[..., :nk] >= threshold).float() * c
        del u
    pd = p if keep is None else p * keep
    o = pd @ v
    outs = [o.to(state["q"].dtype)]
    if case["train"]:
        do = state["grad"].float()
        dv = pd.transpose(-1, -2) @ do
        dp = do @ v.transpose(-1, -2)
        if keep is not None:
            dp = dp * keep
        ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True))
        dq = (ds @ k) * scale
        dk = (ds.transpose(-1, -2) @ q) * scale
        dk, dv = (g.reshape(b, hk, hq // hk, nk, d).sum(dim=2) for g in (dk, dv))
        outs += [g.to(o_.dtype) for g, o_ in ((dq, state["q"]), (dk, state["k"]), (dv, state["v"]))]
    return outs


def _rotate(t, cos, sin):
    n = 2 * cos.shape[-1]
    x, rest = t[..., :n], t[..., n:]
    even, odd = x[..., 0::2], x[..., 1::2]
    y = torch.stack((even * cos - odd * sin, odd * cos + even * sin), dim=-1).flatten(-2)
    return torch.cat((y, rest), dim=-1)


def _plain_rotary(state):
    t = state["t"]
    parts, at = [], 0
    for axis, width in enumerate(state["sections"]):
        parts.append(state["positions"][..., axis, None].double() * state["freqs"][at : at + width].double())
        at += width
    angle = torch.cat(parts, dim=-1)[:, None]  # far positions: the angle needs 64 bits, its sine does not
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    outs = [_rotate(t.float(), cos, sin).to(t.dtype)]
    if state["case"]["train"]:
        outs.append(_rotate(state["grad"].float(), cos, -sin).to(t.dtype))
    return outs


# ------------------------------------------------------------------------------------------------------- run
def _own(state):
    from pymsst_b200.cross_attention import cross_attention, rotary_axes
    from pymsst_b200.dropout import dropout, gelu_dropout

    case = state["case"]
    kind = case["kind"]
    if kind == "dropout":
        leaves = [state["x"]] + ([state["residual"]] if case["residual"] else [])
        y = dropout(state["x"], case["p"], state["key"], state["site"], residual=state.get("residual"))
    elif kind == "gelu_dropout":
        leaves = [state["x"]]
        y = gelu_dropout(state["x"], case["p"], state["key"], state["site"])
    elif kind == "attention":
        leaves = [state["q"], state["k"], state["v"]]
        y = cross_attention(*leaves, key_lengths=state["lengths"], dropout_p=case["p"],
                            key=state["key"] if case["p"] > 0 else None, site=state["site"])
    else:
        leaves = [state["t"]]
        y = rotary_axes(state["t"], state["positions"], state["freqs"], state["sections"])
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, state["grad"])]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        kind = state["case"]["kind"]
        if kind == "attention":
            return _plain_attention(state)
        return _plain_rotary(state) if kind == "rotary" else _plain_dropout(state)


# ----------------------------------------------------------------------------------------------------- exact
def _mul32(a, m):
    """High and low words of the 64-bit product of 32-bit numbers, from 16-bit limbs."""
    a0, a1, m0, m1 = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
    low = a0 * m0
    mid = a1 * m0 + (low >> 16)
    mid2 = a0 * m1 + (mid & 0xFFFF)
    return a1 * m1 + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | (low & 0xFFFF)


def _bits(counter, seed, site):
    """Philox4x32, seven rounds, on a list of four equal-shaped word tensors: eight 16-bit numbers behind them."""
    key = [seed % 2**32, (seed >> 32) % 2**32 ^ site]
    x = list(counter)
    for r in range(7):
        hi0, lo0 = _mul32(x[0], 0xD2511F53)
        hi1, lo1 = _mul32(x[2], 0xCD9E8D57)
        x = [hi1 ^ x[1] ^ ((key[0] + r * 0x9E3779B9) % 2**32), lo1,
             hi0 ^ x[3] ^ ((key[1] + r * 0xBB67AE85) % 2**32), lo0]
    out = torch.empty(*x[0].shape, 4, 2, dtype=torch.int64, device=x[0].device)
    for i, w in enumerate(x):
        out[..., i, 0] = w % 65536
        out[..., i, 1] = w // 65536
    return out.flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    dev = next(v.device for v in state.values() if isinstance(v, torch.Tensor))
    if kind == "rotary":
        pos, freqs = state["positions"].double(), state["freqs"].double()
        axis = torch.repeat_interleave(torch.arange(len(state["sections"]), device=dev),
                                       torch.tensor(state["sections"], device=dev))
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=dev), pos[..., axis] * freqs)[:, None]

        def rotate(t, by):
            t = t.detach().double()
            n = 2 * by.shape[-1]
            z = torch.view_as_complex(t[..., :n].reshape(*t.shape[:-1], -1, 2).contiguous())
            return torch.cat((torch.view_as_real(z * by).flatten(-2), t[..., n:]), dim=-1)

        outs = [rotate(state["t"], turn)]
        return outs + [rotate(state["grad"], turn.conj())] if case["train"] else outs
    seed_word, step = (int(v) for v in state["key"].tolist())
    threshold, c = _threshold(case["p"])
    if kind != "attention":
        x = state["x"].detach().double()
        g = torch.arange(-(-x.numel() // 8), device=dev)
        words = [g % 2**32, g // 2**32, torch.full_like(g, 2**32 - 1), torch.full_like(g, step % 2**32)]
        mult = (_bits(words, seed_word, state["site"]).flatten()[: x.numel()] >= threshold).double() * c
        mult = mult.reshape(x.shape)
        normal = torch.distributions.Normal(torch.zeros((), dtype=torch.float64, device=dev), 1.0)
        gelu = kind == "gelu_dropout"
        y = mult * (x * normal.cdf(x) if gelu else x)
        if case["residual"]:
            y = y + state["residual"].detach().double()
        outs = [y]
        if case["train"]:
            grad = state["grad"].double()
            slope = normal.cdf(x) + x * torch.exp(normal.log_prob(x)) if gelu else 1.0
            outs.append(mult * slope * grad)
            if case["residual"]:
                outs.append(grad)
        return outs
    q, k, v = (state[n].detach() for n in "qkv")
    b, hq, nq, d = q.shape
    hk, nk = k.shape[1], k.shape[2]
    lengths = [nk] * b if state["lengths"] is None else state["lengths"].tolist()
    outs = [torch.zeros(t.shape, dtype=torch.float64, device=dev) for t in ((q, q, k, v) if case["train"] else (q,))]
    query = torch.arange(nq, device=dev)[:, None]
    for i in range(b):
        n = lengths[i]
        if n == 0:
            continue
        group = torch.arange(-(-n // 8), device=dev)[None]
        for h in range(hq):
            kv = h * hk // hq
            qi, ki, vi = q[i, h].double(), k[i, kv, :n].double(), v[i, kv, :n].double()
            if case["train"]:
                for t in (qi, ki, vi):
                    t.requires_grad_()
            prob = torch.softmax(qi @ ki.t() / math.sqrt(d), dim=-1)
            if case["p"] > 0:
                words = torch.broadcast_tensors(group, query, torch.full_like(query, i * hq + h),
                                                torch.full_like(query, step % 2**32))
                u = _bits(words, seed_word, state["site"]).flatten(-2)[:, :n]
                prob = prob * ((u >= threshold).double() * c)
            o = prob @ vi
            outs[0][i, h] = o.detach()
            if case["train"]:
                gq, gk, gv = torch.autograd.grad(o, (qi, ki, vi), state["grad"][i, h].double())
                outs[1][i, h] = gq
                outs[2][i, kv, :n] += gk
                outs[3][i, kv, :n] += gv
    return outs
