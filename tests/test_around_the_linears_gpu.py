"""Embedding, norms around a block and gradient clipping together, as a training step has them around converted
linears; under hooks, checkpoints, tracing and graph capture; and with more elements than 32 bits count."""
import math

import pytest
import torch
import torch.nn as nn

from tests.test_converter_gpu import _convert as _convert_with
from torchtitan_amd import ops
from torchtitan_amd.gradients import clip_grad_norm_
from torchtitan_amd.modules import Embedding, FeedForward, Linear, ResidualRMSNorm, residual_rms_norm, scaled_embedding
from torchtitan_amd.rl.loss import token_log_probs

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


class Model(nn.Module):
    """Two feed-forward blocks with norms on both sides and a gate, between embedding and head."""

    def __init__(self, vocab=700, dim=256, hidden=512):
        super().__init__()
        self.tokens = Embedding.Config(scale=math.sqrt(dim), padding_idx=0).build(num_embeddings=vocab, embedding_dim=dim)
        self.blocks = nn.ModuleList(FeedForward.Config(hidden_dim=hidden).build(dim=dim) for _ in range(2))
        seam = lambda **kw: ResidualRMSNorm.Config(**kw).build(dim=dim)
        self.first = seam()
        self.seams = nn.ModuleList([seam(post_norm=True, gate=True, gate_init=0.5), seam(post_norm=True, residual_scale=0.7)])
        self.head = Linear.Config().build(in_features=dim, out_features=vocab)

    def init(self, seed):
        g = torch.Generator(device=self.head.weight.device).manual_seed(seed)
        with torch.no_grad():
            for name, p in self.named_parameters():
                p.normal_(0.0, 0.05, generator=g)
                if "seam" in name or "first" in name:
                    p.add_(1.0)

    def forward(self, ids):
        x = self.tokens(ids)
        stream, normed = self.first(torch.zeros_like(x), x)
        for block, seam in zip(self.blocks, self.seams):
            stream, normed = seam(block(normed), stream)
        return self.head(normed)


class InTorchOps:
    """The model's operators replaced by the formulas in torch operations, in the parameters' type."""

    def __enter__(self):
        import torchtitan_amd.modules.embedding as e
        import torchtitan_amd.modules.norm as n

        self.kept = e.scaled_embedding, n.residual_rms_norm

        def norm(h, r, *, post_weight, gate, pre_weight, residual_scale, eps):
            return n._in_torch_ops(h, r, post_weight, gate, pre_weight, residual_scale, eps)

        e.scaled_embedding = lambda ids, w, scale, padding_idx: e._in_torch_ops(ids, w, scale, padding_idx, 0, w.dtype)
        n.residual_rms_norm = norm
        self.modules = e, n

    def __exit__(self, *_):
        self.modules[0].scaled_embedding, self.modules[1].residual_rms_norm = self.kept


def _ids(device, seed, shape=(4, 64), vocab=700):
    g = torch.Generator(device=device).manual_seed(seed)
    ids = torch.randint(1, vocab, shape, generator=g, device=device)
    ids[:, -9:] = 0  # padding
    return ids


def _step(model, ids):
    """(loss, gradients by name) of the next tokens' log-probabilities."""
    model.zero_grad(set_to_none=True)
    logits = model(ids)
    target = ids.roll(-1, 1).reshape(-1)
    loss = -token_log_probs(logits.reshape(-1, logits.shape[-1]), target).mean()
    loss.backward()
    return loss.detach(), {n: p.grad for n, p in model.named_parameters()}


def test_a_training_step_equals_the_formulas(device):
    """In float32, against the same model with the formulas in torch operations in float64.  Every value on the way is a
    sum of at most 700 terms of its like and passes six such steps each way, errors of some hundred U in all (U =
    2^-24); products of what is off by that: 1e-4 of a gradient's largest value."""
    model = Model().to(device)
    model.init(1)
    ids = _ids(device, 1)
    loss, grads = _step(model, ids)
    twin = Model().to(device).double()
    twin.load_state_dict(model.state_dict())
    with InTorchOps():
        want_loss, want = _step(twin, ids)
    assert abs(float(loss) - float(want_loss)) <= 1e-5 * abs(float(want_loss))
    for name, g in grads.items():
        assert (g.double() - want[name]).abs().max() <= 1e-4 * want[name].abs().max(), name
    norm = clip_grad_norm_(model.parameters(), 0.01)
    exact = math.sqrt(sum(float(g.square().sum()) for g in want.values()))
    assert abs(float(norm) - exact) <= 1e-4 * exact and exact > 0.01
    clipped = math.sqrt(sum(float(p.grad.double().square().sum()) for p in model.parameters()))
    assert abs(clipped - 0.01 * exact / (exact + 1e-6)) <= 1e-6 * 0.01


def _converted(device):
    model = Model()
    _convert_with(model, ["blocks"])
    model.to(device).to(BF)
    model.init(2)
    return model


def test_a_training_step_of_a_converted_model(device):
    """bf16 with MXFP8 blocks: the same bits on every run; clipped to its limit but for bf16's rounding."""
    model, ids = _converted(device), _ids(device, 2)
    loss, grads = _step(model, ids)
    grads = {n: g.clone() for n, g in grads.items()}
    again, twice = _step(model, ids)
    assert torch.equal(loss, again) and all(torch.equal(g, twice[n]) for n, g in grads.items())
    assert all(g.isfinite().all() and g.any() for g in grads.values())
    assert not grads["tokens.weight"][0].any()  # padding
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads.values()))
    norm = clip_grad_norm_(model.parameters(), exact / 3)
    assert abs(float(norm) - exact) <= 1e-6 * exact
    clipped = math.sqrt(sum(float(p.grad.double().square().sum()) for p in model.parameters()))
    assert abs(clipped - exact / 3) <= exact / 3 * (2.0 ** -8 + 1e-5)  # (every value off by at most half a step)


def test_a_captured_training_step_replays(device):
    model, ids = _converted(device), _ids(device, 3)
    batches = [_ids(device, 10 + k) for k in range(3)]
    eager = []
    for batch in batches:
        _, grads = _step(model, batch)
        norm = clip_grad_norm_(model.parameters(), 0.02)
        eager.append([norm.clone()] + [g.clone() for g in grads.values()])
        del grads, norm
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(model, ids)
        clip_grad_norm_(model.parameters(), 0.02)
    torch.cuda.current_stream().wait_stream(side)
    model.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model(ids)
        loss = -token_log_probs(logits.reshape(-1, logits.shape[-1]), ids.roll(-1, 1).reshape(-1)).mean()
        loss.backward()
        norm = clip_grad_norm_(model.parameters(), 0.02)
    del logits, loss
    for _ in range(2):
        for batch, want in zip(batches, eager):
            ids.copy_(batch)
            graph.replay()
            torch.cuda.synchronize()
            got = [norm] + [p.grad for p in model.parameters()]
            assert torch.randn(1 << 20, device=device).sum().isfinite()  # eager work between replays
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def _operands(device, shape=(3, 40, 320), dtype=BF, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    n = lambda s: torch.randn(s, generator=g, device=device).to(dtype).requires_grad_(True)
    return [n(shape), n(shape), n(shape[-1:]), n((shape[0], 1, shape[-1])), n(shape[-1:])]


def _norm(t):
    return residual_rms_norm(t[0], t[1], post_weight=t[2], gate=t[3], pre_weight=t[4], residual_scale=0.5)


def test_saved_tensors_that_hooks_replace(device):
    """Copies on the host and back, copies with other strides: the same gradients; tensors that do not fit: an error."""
    ids = torch.randint(0, 50, (7, 9), device=device)
    weight = torch.randn((50, 24), device=device).to(BF).requires_grad_(True)
    operands = _operands(device)

    def run(pack, unpack):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = [scaled_embedding(ids, weight, 2.0), *_norm(operands)]
        return torch.autograd.grad([t.float().square().sum() for t in out], [weight, *operands])

    want = run(lambda t: t, lambda t: t)

    def strided(t):
        wide = torch.empty((*t.shape, 2), dtype=t.dtype, device=t.device)
        wide[..., 0] = t
        return wide[..., 0]

    for got in (run(lambda t: t.cpu(), lambda t: t.to(device)), run(strided, lambda t: t)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for spoil in (lambda t: t.cpu(), lambda t: t[..., :1] if t.dim() > 1 else t):
        with pytest.raises(RuntimeError):
            run(lambda t: t, spoil)


def test_checkpointed_seams(device):
    from torch.utils.checkpoint import checkpoint

    operands = _operands(device, seed=1)
    want = torch.autograd.grad([t.float().square().sum() for t in _norm(operands)], operands)
    for reentrant in (False, True):
        out = checkpoint(lambda *t: _norm(t), *operands, use_reentrant=reentrant)
        for t in operands:
            t.grad = None
        sum(t.float().square().sum() for t in out).backward()
        assert all(torch.equal(t.grad, g) for t, g in zip(operands, want))


@pytest.mark.parametrize("native", [True, False])
def test_gradients_cannot_be_differentiated_again(device, native, monkeypatch):
    if not native:
        monkeypatch.setattr(ops, "native_rows", lambda t: False)
    operands = _operands(device, seed=2)
    weight = torch.randn((50, 24), device=device, requires_grad=True)
    ids = torch.randint(0, 50, (7, 9), device=device)
    for out, leaf in ((_norm(operands)[1].float(), operands[0]), (scaled_embedding(ids, weight), weight)):
        (grad,) = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentia"):
            grad.float().square().sum().backward()


def test_native_calls_and_general_path_agree(device, monkeypatch):
    operands = _operands(device, (6, 17, 1030), seed=3)
    weight = torch.randn((90, 130), device=device).to(BF).requires_grad_(True)
    ids = torch.randint(-3, 95, (5, 70), device=device)
    grads = [torch.randn((300, 41), device=device).to(BF), torch.randn(7, device=device)]

    def everything():
        out = [scaled_embedding(ids, weight, 3.0, padding_idx=4, dtype=torch.float32), *_norm(operands)]
        mine = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
        for p, g in zip(mine, grads):
            p.grad = g.clone()
        norm = clip_grad_norm_(mine, 0.5)
        return [t.detach() for t in out] + list(torch.autograd.grad([t.float().square().sum() for t in out], [weight, *operands])) + [
            norm] + [p.grad for p in mine]

    native = everything()
    monkeypatch.setattr(ops, "native_rows", lambda t: False)
    assert all(torch.equal(a, b) for a, b in zip(native, everything()))


def test_traced_operators_equal_eager(device):
    import torch._dynamo

    model, ids = _converted(device), _ids(device, 4, (4, 64))
    _, want = _step(model, ids)
    want = {n: g.clone() for n, g in want.items()}
    torch._dynamo.reset()
    try:
        model.forward = torch.compile(model.forward, backend="aot_eager", fullgraph=True)
        _, got = _step(model, ids)
        for name, g in got.items():
            assert torch.equal(g, want[name]), name
        with torch.no_grad():
            assert torch.equal(model(ids), _plain_forward(model, ids))
    finally:
        del model.forward
        torch._dynamo.reset()


def _plain_forward(model, ids):
    return Model.forward(model, ids)


def test_more_elements_than_32_bits_count(device):
    """The last rows of matrices of 2^31 elements and more, against the operators on those rows alone."""
    rows, dim, last = 530000, 4100, 500  # 2.17e9 elements
    weight = torch.empty((rows, dim), dtype=BF, device=device)
    weight[-last:] = torch.randn((last, dim), device=device).to(BF)
    ids = torch.arange(rows - last, rows, device=device).flip(0).repeat(2)
    out = ops.embedding_fwd(ids, weight, 2.0)
    assert torch.equal(out[:last], (weight[-last:].float() * 2).to(BF).flip(0))
    dout = torch.randn((2 * last, dim), device=device).to(BF)
    for tokens in (ids, torch.cat([ids, torch.full((9000,), -1, device=device)])):  # placed in one launch, and by radix passes
        d = torch.cat([dout, dout.new_ones((tokens.numel() - 2 * last, dim))])
        grad = ops.embedding_bwd(tokens, d, rows)
        both = dout[:last].float() + dout[last:].float()
        assert torch.equal(grad[-last:], both.to(BF).flip(0)) and not grad[: rows - last].any()
        del grad, d
    h, r = weight, torch.zeros_like(weight)
    h[: rows - last] = 1
    r[-last:] = torch.randn((last, dim), device=device).to(BF)
    post, gate, pre = (torch.rand(dim, device=device).to(BF) for _ in range(3))
    stream, normed, rstd = ops.residual_norm(h, r, post, gate[None], pre, 0.5, 1e-5, want_rstd=True)
    alone = ops.residual_norm(h[-last:], r[-last:], post, gate[None], pre, 0.5, 1e-5, want_rstd=True)
    assert torch.equal(stream[-last:], alone[0]) and torch.equal(normed[-last:], alone[1]) and torch.equal(rstd[:, -last:], alone[2])
    dh, dr, *_ = ops.residual_norm_bwd(h, r, post, gate[None], pre, 0.5, rstd, stream, normed)
    dh1, dr1, *_ = ops.residual_norm_bwd(h[-last:], r[-last:], post, gate[None], pre, 0.5, alone[2], alone[0], alone[1])
    assert torch.equal(dh[-last:], dh1) and torch.equal(dr[-last:], dr1)
    del dh, dr, stream, normed, r
    h[: rows - last] = 0
    norm = ops.grad_norm([h])
    tail = float(h[-last:].double().square().sum()) ** 0.5
    assert abs(float(norm) - tail) <= 2.0 ** -23 * tail
    before = h[-last:].clone()
    ops.grad_scale_([h], norm, float(norm) / 4)
    factor = (float(norm) / 4) / (float(norm) + 1e-6)
    assert ((h[-last:].double() - before.double() * factor).abs() <= before.double().abs() * 2.0 ** -8).all()


def test_negated_views(device):
    """Views whose memory holds the negated values: read as the values that they stand for, or refused."""
    neg = torch._neg_view
    operands = [t.detach() for t in _operands(device, seed=5)]
    dense = [(-t).requires_grad_(True) for t in operands]
    views = [neg(t).requires_grad_(True) for t in operands]
    g = torch.randn(operands[0].shape, device=device).to(BF)
    ids = torch.randint(0, 3, (40,), device=device)
    d = torch.randn((40, 320), device=device).to(BF)
    for into, of in ((lambda t: t, lambda t: t), (lambda t: -t, neg)):
        want = torch.autograd.grad(_norm(dense), dense, [into(g), into(g)])
        for got in (torch.autograd.grad(_norm(dense), dense, [of(g), of(g)]), torch.autograd.grad(_norm(views), views, [of(g), of(g)])):
            assert all((a - b).abs().max() <= 2.0 ** -7 * b.abs().max() for a, b in zip(got, want))  # (torch operations round alike)
        table, seen = dense[0][0].detach().requires_grad_(True), neg(operands[0][0]).requires_grad_(True)
        a, b = scaled_embedding(ids, table, 2.0), scaled_embedding(ids, seen, 2.0)
        assert torch.equal(a, b)
        assert torch.equal(torch.autograd.grad(a, table, into(d))[0], torch.autograd.grad(scaled_embedding(ids, table, 2.0), table, of(d))[0])
    assert torch.equal(ops.embedding_fwd(ids, neg(operands[0][0])), -ops.embedding_fwd(ids, operands[0][0]))
    with pytest.raises(ValueError):
        ops.grad_norm([neg(operands[0])])
    p = nn.Parameter(torch.zeros(8, device=device))
    p.grad = neg(torch.ones(8, device=device))
    with pytest.raises(RuntimeError):
        clip_grad_norm_([p], 0.1)


def test_batched_gradients_are_refused(device):
    operands = _operands(device, seed=6)
    stream, normed = _norm(operands)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(stream, operands[0], torch.ones((2, *stream.shape), dtype=BF, device=device), is_grads_batched=True)
    weight = torch.randn((9, 16), device=device, requires_grad=True)
    out = scaled_embedding(torch.zeros(5, dtype=torch.int64, device=device), weight)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, weight, torch.ones((2, *out.shape), device=device), is_grads_batched=True)


def test_nothing_outlives_its_graph(device):
    operands = _operands(device, (4, 512, 1024), seed=7)
    ids = torch.randint(0, 100, (4, 512), device=device)
    weight = torch.randn((100, 1024), device=device).to(BF).requires_grad_(True)
    for _ in range(3):
        before = torch.cuda.memory_allocated()
        out = [*_norm(operands), scaled_embedding(ids, weight)]
        torch.autograd.grad([t.sum() for t in out], [*operands, weight])
        out = [*_norm(operands), scaled_embedding(ids, weight)]  # (and one without a backward)
        del out
        assert torch.cuda.memory_allocated() == before


def test_two_graphs_and_two_streams(device):
    """Two captured passes replayed in turn and out of turn, and two streams at work at once: no shared workspace."""
    sets = []
    for seed in (8, 9):
        operands = _operands(device, (5, 700, 512), seed=seed)
        ids = torch.randint(0, 3000, (9000,), device=device, generator=torch.Generator(device=device).manual_seed(seed))
        d = torch.randn((9000, 96), device=device).to(BF)
        sets.append(([t.detach() for t in operands], ids, d))

    def work(s):
        (h, r, post, gate, pre), ids, d = s
        h2, r2 = h.view(-1, 512), r.view(-1, 512)
        stream, normed, rstd = ops.residual_norm(h2, r2, post, gate.view(-1, 512), pre, 0.5, 1e-5, True)
        grads = ops.residual_norm_bwd(h2, r2, post, gate.view(-1, 512), pre, 0.5, rstd, stream, normed)
        table = ops.embedding_bwd(ids, d, 3000)
        scaled = [g.clone() for g in grads]
        norm = ops.grad_norm(scaled)
        ops.grad_scale_(scaled, norm, 0.1)
        return [stream, normed, *grads, table, norm, *scaled]

    want = [[t.clone() for t in work(s)] for s in sets]
    graphs, outs = [], []
    for s in sets:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work(s))
        graphs.append(graph)
    for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for k in order:
            graphs[k].replay()
        torch.cuda.synchronize()
        assert torch.randn(1 << 20, device=device).sum().isfinite()
        for got, expected in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, expected))
    streams = [torch.cuda.Stream() for _ in sets]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(work(s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_more_rows_than_two_a_workgroup_reach(device):
    """2^29 rows of 16 lanes each, two a lane: 2^32 lanes, one more than a launch has.  The first and last rows against the
    operator on them alone."""
    rows, dim, few = (1 << 29) + 5, 8, 4099
    h, r = (torch.zeros((rows, dim), dtype=BF, device=device) for _ in range(2))
    post, pre = (1 + torch.rand(dim, device=device).to(BF) for _ in range(2))
    for part in (slice(0, few), slice(rows - few, rows)):
        h[part], r[part] = (torch.randn((few, dim), device=device).to(BF) for _ in range(2))
    stream, normed, rstd = ops.residual_norm(h, r, post, None, pre, 0.5, 1e-5, want_rstd=True)
    for part in (slice(0, few), slice(rows - few, rows)):
        alone = ops.residual_norm(h[part], r[part], post, None, pre, 0.5, 1e-5, want_rstd=True)
        assert torch.equal(stream[part], alone[0]) and torch.equal(normed[part], alone[1]) and torch.equal(rstd[:, part], alone[2])
    assert not stream[few:-few:4097].any()
    del h, r, stream, normed, rstd
    torch.cuda.empty_cache()


@pytest.mark.parametrize("native", [True, False])
def test_a_penalty_on_a_gradient_is_refused_whatever_it_is_formed_from(device, native, monkeypatch):
    """The norms' operands are in their gradients: a penalty beside a loss is an error, not left out, where the outputs'
    gradients are constants too.  A plain sum has none of them in its gradients, and no penalty to lose."""
    if not native:
        monkeypatch.setattr(ops, "native_rows", lambda t: False)
    h, r, post, gate, pre = _operands(device, seed=10)
    for weights, out in ((dict(pre_weight=pre), 1), (dict(post_weight=post), 0), (dict(gate=gate), 0), (dict(post_weight=post, pre_weight=pre), 0)):
        loss = residual_rms_norm(h, r, **weights)[out].float().sum()
        grads = torch.autograd.grad(loss, [h, *weights.values()], create_graph=True, allow_unused=True)
        for g in grads:
            with pytest.raises(RuntimeError, match="differentia"):
                (loss + g.float().square().sum()).backward(retain_graph=True)
    stream, _ = residual_rms_norm(h, r, residual_scale=0.5)
    dh, dr = torch.autograd.grad(stream.float().sum(), [h, r], create_graph=True)
    assert not dh.requires_grad and (dr == 0.5).all()
    for use in (dict(create_graph=True), dict()):  # and a backward that nobody differentiates goes through
        h.grad = None
        residual_rms_norm(h, r, pre_weight=pre)[1].float().sum().backward(**use)
        assert h.grad.isfinite().all() and h.grad.requires_grad == bool(use)
    h.grad = None
