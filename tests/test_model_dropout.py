"""Models whose dropout comes from a generator, and the new operators in a row as a block uses them."""
from __future__ import annotations

import contextlib
import gc
import math
import weakref

import pytest
import torch

from oracle import context_ref as ref
from pymsst_b200 import _native as nat
from pymsst_b200 import config as cfg
from pymsst_b200 import dropout as dropout_module
from pymsst_b200 import synthetic
from pymsst_b200.cross_attention import cross_attention, rotary_axes
from pymsst_b200.dropout import DropoutGenerator, dropout, gelu_dropout
from pymsst_b200.roformer import Attention, FeedForward
from pymsst_b200.train import Trainer
from tests.model_configs import CONFIG0_BSR, TINY_BSR

DROP = dict(attn_dropout=0.1, ff_dropout=0.2)
TINY_LOSS = dict(TINY_BSR, multi_stft_resolutions_window_sizes=(128, 64), multi_stft_hop_size=16)


def _model(kwargs, device, **extra):
    torch.manual_seed(0)
    return cfg.build_model("bs_roformer", **dict(kwargs, **DROP, **extra)).to(device)


def test_sites_are_distinct():
    model = cfg.build_model("bs_roformer", **dict(TINY_BSR, depth=2, **DROP))
    model.set_dropout_generator(None)
    sites = [s for m in model.modules() if isinstance(m, (Attention, FeedForward))
             for s in (m.dropout_site, m.dropout_site + 1)]
    assert len(sites) == len(set(sites)) == 16
    assert model._dropout_key() is None


@pytest.mark.gpu
def test_block_of_the_operators_against_64_bits(cuda_device):
    """Rotary positions of queries and context, attention with dropout, output dropout with the residual sum, GELU with
    dropout: fp32 kernels against the definitions with the same masks, values and gradients.  Every operator is fp32
    with products and sums of at most 128 terms of order one; four of them in a row, their errors amplified by the
    following ones' slopes (below 10 here), stay under 4 x 128 x 2^-24 x 10 = 3e-4."""
    g = torch.Generator().manual_seed(5)
    b, h, nq, nk, d = 2, 4, 9, 21, 16
    seed, step = 77, 3
    x = torch.randn(b, nq, h * d, generator=g)
    ctx = torch.randn(b, nk, h * d, generator=g)
    w = torch.randn(h * d, h * d, generator=g) / math.sqrt(h * d)
    gy = torch.randn(b, nq, h * d, generator=g)
    freqs = torch.tensor([1.0, 0.3, 0.1, 0.7, 0.2])
    pos_q = torch.randint(0, 50, (b, nq, 2), generator=g)
    pos_k = torch.randint(0, 50, (b, nk, 2), generator=g)
    lengths = [nk, 13]
    key = torch.tensor([seed, step], device=cuda_device)

    def run(x, ctx, w, dev):
        q, k = x.reshape(b, nq, h, d).transpose(1, 2), ctx.reshape(b, nk, h, d).transpose(1, 2)
        if dev:
            f = freqs.to(cuda_device)
            q, kr = (rotary_axes(t, p.to(cuda_device), f, [3, 2]) for t, p in ((q, pos_q), (k, pos_k)))
            o = cross_attention(q, kr, k, key_lengths=torch.tensor(lengths, device=cuda_device), dropout_p=0.2, key=key,
                                site=0)
            o = o.transpose(1, 2).reshape(b, nq, h * d)
            y = dropout(o @ w, 0.3, key, 1, residual=x)
            return gelu_dropout(y, 0.1, key, 2)
        q, kr = (ref.rotary_axes(t, p, freqs, [3, 2]) for t, p in ((q, pos_q), (k, pos_k)))
        o = ref.attention(q, kr, k, lengths, None, ref.attention_mult(b, h, nq, nk, 0.2, seed, step, 0))
        o = o.transpose(1, 2).reshape(b, nq, h * d)
        y = x + (o @ w) * ref.dropout_mult(x.numel(), 0.3, seed, step, 1).reshape(x.shape)
        cdf = 0.5 * torch.erfc(-y * 2.0**-0.5)
        return y * cdf * ref.dropout_mult(x.numel(), 0.1, seed, step, 2).reshape(x.shape)

    ours = [t.to(cuda_device).requires_grad_() for t in (x, ctx, w)]
    exact = [t.double().requires_grad_() for t in (x, ctx, w)]
    y, e = run(*ours, True), run(*exact, False)
    assert float((y.detach().double().cpu() - e.detach()).abs().max()) < 3e-4 * float(e.detach().abs().max())
    for a, c in zip(torch.autograd.grad(y, ours, gy.to(cuda_device)), torch.autograd.grad(e, exact, gy.double())):
        assert float((a.double().cpu() - c).abs().max()) < 3e-4 * float(c.abs().max())


@pytest.mark.gpu
def test_no_generator_and_evaluation_are_as_before(cuda_device):
    mix, _ = synthetic.make_batch(2, 256, seed=1)
    mix = mix.to(cuda_device)
    model = _model(TINY_BSR, cuda_device)
    torch.manual_seed(3)
    before = model(mix)
    model.eval()
    plain = model(mix)
    model.set_dropout_generator(DropoutGenerator(1, cuda_device))
    assert torch.equal(plain, model(mix))
    assert model.dropout_generator.state_dict() == {"seed": 1, "step": 0}
    model.train()
    assert not torch.equal(before, model(mix))
    model.set_dropout_generator(None)
    torch.manual_seed(3)
    assert torch.equal(before, model(mix))


@pytest.mark.gpu
@pytest.mark.parametrize("kwargs,length,amp", [(TINY_LOSS, 256, None), (CONFIG0_BSR, 16384, torch.bfloat16)])
def test_recomputed_transformers_draw_the_same_masks(cuda_device, kwargs, length, amp):
    """The same kernels on the same inputs and masks: loss and gradients to the last bits of their sums."""
    mix, tgt = (t.to(cuda_device) for t in synthetic.make_batch(1, length, seed=1))
    results = []
    for recompute in (False, True):
        model = _model(kwargs, cuda_device, use_torch_checkpoint=recompute)
        model.set_dropout_generator(DropoutGenerator(11, cuda_device))
        with torch.autocast("cuda", dtype=amp or torch.bfloat16, enabled=amp is not None):
            loss = model(mix, tgt)
        loss.backward()
        results.append((float(loss.detach()), {n: p.grad for n, p in model.named_parameters() if p.grad is not None}))
    (loss_a, grads_a), (loss_b, grads_b) = results
    assert loss_a == loss_b and grads_a.keys() == grads_b.keys()
    for name, ga in grads_a.items():
        scale = float(ga.abs().max())
        assert float((ga - grads_b[name]).abs().max()) <= 1e-5 * scale, name


@pytest.mark.gpu
def test_types_share_their_masks(cuda_device):
    """bf16 autocast against fp32 with one key: the masks go by element, so the stems agree as they do without dropout
    (2e-2 relative, the package's bf16 bound)."""
    mix, _ = synthetic.make_batch(1, 16384, seed=2)
    mix = mix.to(cuda_device)
    model = _model(CONFIG0_BSR, cuda_device)
    gen = DropoutGenerator(5, cuda_device)
    model.set_dropout_generator(gen)
    with torch.no_grad():
        full = model(mix)
        gen.manual_seed(5)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            half = model(mix)
        other = model(mix)
    assert float((half.float() - full).norm() / full.norm()) < 2e-2
    assert float((other - full).norm() / full.norm()) > 2e-2  # another step, other masks


@pytest.mark.gpu
def test_gradient_along_a_direction(cuda_device):
    """Central difference of a smooth function of the fp32 stems with the key held: L is a sum of 512 products, its
    rounding about 2^-24 x sqrt(512) x 10 = 1.4e-5 of its terms' size; over 2 h = 0.02 that is 7e-4 of |L'| ~ 1, and
    h^2 adds 1e-4 times the third derivative.  2 % leaves a factor ten."""
    mix, _ = synthetic.make_batch(1, 256, seed=1)
    mix = mix.to(cuda_device)
    model = _model(TINY_BSR, cuda_device)
    gen = DropoutGenerator(9, cuda_device)
    model.set_dropout_generator(gen)
    torch.manual_seed(1)
    weight = torch.randn_like(model(mix))

    def value():
        gen.manual_seed(9)
        return (model(mix).double() * weight.double()).sum()

    value().backward()
    params = [p for p in model.parameters() if p.grad is not None]
    dirs = [p.grad / p.grad.norm().clamp_min(1e-12) for p in params]
    slope = sum(float((p.grad.double() * d.double()).sum()) for p, d in zip(params, dirs))
    h = 1e-2 / math.sqrt(len(params))
    out = []
    with torch.no_grad():
        for sign in (1, -1):
            for p, d in zip(params, dirs):
                p.add_(d, alpha=sign * h)
            out.append(float(value()))
            for p, d in zip(params, dirs):
                p.sub_(d, alpha=sign * h)
    assert abs((out[0] - out[1]) / (2 * h) - slope) < 2e-2 * abs(slope)


@pytest.mark.gpu
@pytest.mark.parametrize("recompute", [False, True])
def test_captured_training_step_draws_new_masks_each_replay(cuda_device, recompute):
    """A captured run and an uncaptured one with generators of one seed see the same masks step by step: their losses
    agree to what fp32 sums in another order leave (1e-4 relative over three Adam steps); a run of another seed does
    not."""
    mix, tgt = (t.to(cuda_device) for t in synthetic.make_batch(1, 256, seed=1))
    losses = []
    for graph, seed in ((False, 4), (True, 4), (True, 8)):
        model = _model(TINY_LOSS, cuda_device, use_torch_checkpoint=recompute)
        model.set_dropout_generator(DropoutGenerator(seed, cuda_device))
        trainer = Trainer(model, lr=1e-3, cuda_graph=graph, device=cuda_device)
        losses.append([float(trainer.step(mix, tgt)) for _ in range(3)])
        assert model.dropout_generator.state_dict() == {"seed": seed, "step": 3}
        trainer.close()
        del trainer, model
    eager, captured, other = losses
    assert len(set(captured)) == 3
    for a, b, c in zip(eager, captured, other):
        assert abs(a - b) <= 1e-4 * abs(a)
        assert abs(a - c) > 1e-4 * abs(a)


def _operator_calls(device):
    """One call of each operator without a gradient to any input: the call, and the inputs that are numbers."""
    def rand(*shape):
        return torch.randn(*shape, device=device)

    key = torch.tensor([1, 2], device=device)
    q, k, v = rand(1, 2, 3, 8), rand(1, 1, 5, 8), rand(1, 1, 5, 8)
    return {
        "dropout": (lambda x, r: dropout(x, 0.5, key, residual=r), (rand(16), rand(16))),
        "dropout_without_residual": (lambda x: dropout(x, 0.5, key), (rand(16),)),
        "gelu_dropout": (lambda x: gelu_dropout(x, 0.5, key), (rand(16),)),
        "cross_attention": (cross_attention, (q, k, v)),
        "rotary_axes": (lambda t, pos, f: rotary_axes(t, pos, f, [2, 2]), (q, rand(3, 2), rand(4))),
    }


def _refuses_tangents(device):
    forward_ad = torch.autograd.forward_ad
    for name, (call, inputs) in _operator_calls(device).items():
        call(*inputs)
        with forward_ad.dual_level():
            call(*inputs)  # no tangent among the inputs
            for i in range(len(inputs)):
                duals = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(inputs)]
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
                        call(*duals)
                        pytest.fail(f"{name}: input {i}'s tangent is gone without an error")


def test_forward_mode_tangents_are_refused(monkeypatch):
    """Nothing may drop a tangent; the launches are replaced by copies, as no GPU is needed to see which way a call
    takes."""
    from pymsst_b200 import cross_attention as attention_module

    monkeypatch.setattr(nat, "require_cuda", lambda *t, name: t[0].device)
    monkeypatch.setattr(dropout_module, "_dropout", lambda x, *rest: x.clone())
    monkeypatch.setattr(dropout_module, "_gelu_dropout", lambda x, *rest: x.clone())
    monkeypatch.setattr(attention_module, "_attention_forward", lambda q, *rest: (q.clone(), q.new_zeros(1)))
    monkeypatch.setattr(attention_module, "_rotary", lambda t, *rest: t.clone())
    _refuses_tangents("cpu")


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused_on_the_device(cuda_device):
    _refuses_tangents(cuda_device)


class _Stub(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.lin = torch.nn.Linear(4, 4)
        self.dropout_generator = None

    def forward(self, mix, target):
        return (self.lin(mix) - target).abs().mean()


def test_exchanged_generator_captures_the_step_again(monkeypatch):
    """Host logic of the captured step on the CPU, the capture and its replay replaced by counters."""
    trainer = Trainer(_Stub(), device=torch.device("cpu"))
    trainer.cuda_graph = True
    replays = []

    class Graph:
        def replay(self):
            replays.append(self)

    def capture(mixture, target):
        trainer._graph, trainer._static = Graph(), (mixture.clone(), target.clone(), torch.zeros(()))

    monkeypatch.setattr(trainer, "_capture", capture)
    mix = torch.zeros(2, 4)
    seen = []
    first, second = object(), object()
    for generator in (None, None, first, first, second, None):
        trainer.model.dropout_generator = generator
        trainer.step(mix, mix)
        seen.append(replays[-1])
    assert seen[0] is seen[1] and seen[2] is seen[3]
    assert len({id(g) for g in seen}) == 4


def test_captured_state_outlives_its_generator(monkeypatch):
    """A key drawn while a stream captures leaves the state's address in the graph; drawn otherwise it does not."""
    monkeypatch.setattr(nat, "require_cuda", lambda *t, name: t[0].device)
    monkeypatch.setattr(nat, "stream_handle", lambda device: 0)
    monkeypatch.setattr(nat, "call", lambda *args: None)
    monkeypatch.setattr(dropout_module, "on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(dropout_module, "_captured_states", [])
    for capturing in (False, True):
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
        gen = DropoutGenerator(1, "cpu")
        gen.next_key()
        gen.next_key()
        state = weakref.ref(gen.state)
        del gen
        gc.collect()
        assert (state() is not None) == capturing
    assert len(dropout_module._captured_states) == 1


@pytest.mark.gpu
def test_replays_write_no_released_memory(cuda_device):
    """The generator of a captured forward is dropped and blocks of its state's size are handed out again: replays leave
    them alone and go on drawing new masks."""
    gen = DropoutGenerator(6, cuda_device)
    x = torch.ones(4096, device=cuda_device)
    dropout(x, 0.5, gen.next_key())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dropout(x, 0.5, gen.next_key())
    del gen
    gc.collect()
    others = [torch.zeros(2, dtype=torch.int64, device=cuda_device) for _ in range(256)]
    masks = []
    for _ in range(3):
        graph.replay()
        masks.append(y.clone())
    assert not any(bool(t.any()) for t in others)
    for replay, mask in enumerate(masks):
        assert torch.equal(mask.cpu().double(), ref.dropout_mult(x.numel(), 0.5, 6, 1 + replay, 0))


@pytest.mark.gpu
def test_captured_trainer_follows_an_exchanged_generator(cuda_device):
    """Two steps with one generator, two with another, against the same steps uncaptured: equal losses to what fp32 sums
    in another order leave (1e-4 relative over four Adam steps), equal steps of both generators; then none."""
    mix, tgt = (t.to(cuda_device) for t in synthetic.make_batch(1, 256, seed=1))
    losses = []
    for graph in (False, True):
        model = _model(TINY_LOSS, cuda_device)
        trainer = Trainer(model, lr=1e-3, cuda_graph=graph, device=cuda_device)
        run = []
        for seed in (4, 8):
            model.set_dropout_generator(DropoutGenerator(seed, cuda_device))
            run += [float(trainer.step(mix, tgt)) for _ in range(2)]
            assert model.dropout_generator.state_dict() == {"seed": seed, "step": 2}
        losses.append(run)
        model.set_dropout_generator(None)
        last = [float(trainer.step(mix, tgt)) for _ in range(3)]
        assert len(set(last)) == 3 and all(math.isfinite(v) for v in last)
        trainer.close()
    for a, b in zip(*losses):
        assert abs(a - b) <= 1e-4 * abs(a)


def test_relayout_pass_takes_no_step_of_the_generator(monkeypatch):
    """The pass that orders the flat buffers (overlapped all-reduce, one rank here) draws a key; the training steps start
    where the generator was."""
    import torch.distributed as dist

    class Counter:
        def __init__(self):
            self.state = torch.tensor([3, 0])
            self.drawn = []

        def next_key(self):
            self.drawn.append(int(self.state[1]))
            self.state[1] += 1

    class Model(_Stub):
        def forward(self, mix, target):
            self.dropout_generator.next_key()
            return super().forward(mix, target)

    monkeypatch.setattr(dist, "broadcast", lambda tensor, src: None)
    trainer = Trainer(Model(), device=torch.device("cpu"), flat_params=True)
    generator = trainer.model.dropout_generator = Counter()
    trainer._relayout_done = False
    for _ in range(2):
        trainer.step(torch.randn(2, 4), torch.randn(2, 4))
    assert generator.drawn == [0, 0, 1] and generator.state.tolist() == [3, 2]


@pytest.mark.gpu
def test_profiled_replays_take_no_step_of_the_generator(cuda_device):
    mix, tgt = (t.to(cuda_device) for t in synthetic.make_batch(1, 256, seed=1))
    model = _model(TINY_LOSS, cuda_device)
    model.set_dropout_generator(DropoutGenerator(4, cuda_device))
    trainer = Trainer(model, lr=1e-3, cuda_graph=True, device=cuda_device)
    trainer.step(mix, tgt)
    profile = trainer.profile_graph()
    for _ in range(3):
        profile.replay()
    assert model.dropout_generator.state_dict() == {"seed": 4, "step": 1}
    trainer.step(mix, tgt)
    assert model.dropout_generator.state_dict() == {"seed": 4, "step": 2}
    trainer.close()
