"""The operators of a training step around the converted linears, as a user's program calls them.

Token embedding with its gradient, the norms before and after a block with its gate and residual scale,
and the clipping of the gradients by their norm.  Sizes are those of the benchmark, the tests and the
layer shapes they name (model size 4096, 2048 with hidden size 6144, vocabulary 151 936, 147 456 packed
tokens of a policy step) and of counts around them, packed and ragged.

``listed()`` gives the fixed cases, ``draw(rng)`` another one of the same ranges, ``prepare`` what a
program holds before the call, ``run`` one pass -- with ``own`` through the framework's operators, else
in elementary torch operations --, ``work`` the bytes and operations a pass cannot do without, ``exact``
the results in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # A generator's step over a handful of sequences: one token each.  The smallest lookup.
        dict(name="embedding_few_tokens", kind="embedding", train=False, tokens=16, vocab=151936, first=0, rows=151936,
             dim=2048, params="bfloat16", out="bfloat16", scale=1.0, ids="uniform"),
        # A short micro-batch, every sequence padded to the longest: a third of the tokens is padding, which
        # has no gradient.  The gradient of the whole table is written, whatever the tokens.
        dict(name="embedding_train_padded", kind="embedding", train=True, tokens=2003, vocab=151936, first=0, rows=151936,
             dim=2048, params="bfloat16", out="bfloat16", scale=45.25, ids="padded"),
        # One of eight vocabulary shards under tensor parallelism, float32 parameters under autocast to
        # bfloat16: most tokens lie in the other shards.
        dict(name="embedding_train_shard", kind="embedding", train=True, tokens=8192, vocab=151936, first=37984, rows=18992,
             dim=4096, params="float32", out="bfloat16", scale=64.0, ids="skewed"),
        # All packed tokens of one policy step, some tokens far more frequent than others.
        dict(name="embedding_train_packed", kind="embedding", train=True, tokens=147456, vocab=151936, first=0, rows=151936,
             dim=2048, params="bfloat16", out="bfloat16", scale=1.0, ids="skewed"),
        # A generator's step: both norms, gate and residual of one block for 16 tokens.  The smallest norm.
        dict(name="norm_few_tokens", kind="norm", train=False, rows=16, dim=2048, post=True, gate=1, pre=True,
             block="bfloat16", stream="bfloat16", params="bfloat16", scale=1.0),
        # The plain pre-norm block in training, few tokens: residual sum and the next norm.
        dict(name="norm_train_plain_ragged", kind="norm", train=True, rows=3001, dim=4096, post=False, gate=0, pre=True,
             block="bfloat16", stream="bfloat16", params="bfloat16", scale=1.0),
        # Norms on both sides around a residual stream that is kept in float32.
        dict(name="norm_train_float32_stream", kind="norm", train=True, rows=8191, dim=2048, post=True, gate=0, pre=True,
             block="bfloat16", stream="float32", params="float32", scale=1.0),
        # Both norms, a gate per channel and a scaled residual at the benchmark's token count.
        dict(name="norm_train_gated", kind="norm", train=True, rows=16384, dim=4096, post=True, gate=1, pre=True,
             block="bfloat16", stream="bfloat16", params="bfloat16", scale=0.5),
        # The same over all packed tokens of a policy step, with a gate for each of its 16 sequences.
        dict(name="norm_train_sequence_gates", kind="norm", train=True, rows=147456, dim=2048, post=True, gate=16, pre=True,
             block="bfloat16", stream="bfloat16", params="bfloat16", scale=1.0),
        # One layer of a model as small as the tests': a handful of small gradients.  The smallest clipping.
        dict(name="clip_small_layer", kind="clip", layers=1, inner=128, outer=512, vocab=0, params="bfloat16", norm=2.0),
        # One layer's gradients (four attention projections, three of the feed-forward block, four norms).
        dict(name="clip_layer", kind="clip", layers=1, inner=2048, outer=6144, vocab=0, params="bfloat16", norm=2.0),
        # Four layers with embedding and head, float32 master gradients: 3.3 GB.
        dict(name="clip_model_float32", kind="clip", layers=4, inner=2048, outer=6144, vocab=151936, params="float32", norm=2.0),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["embedding", "embedding", "norm", "norm", "clip"])
    params = rng.choice(["bfloat16", "bfloat16", "float32"])
    if kind == "embedding":
        vocab = _log_uniform(rng, 257, 151936)
        tokens = _log_uniform(rng, 1, 65536)
        rows = vocab if rng.random() < 0.6 else max(1, vocab // rng.choice([2, 3, 8]))
        return dict(kind=kind, train=rng.random() < 0.75, tokens=tokens, vocab=vocab, first=rng.randrange(vocab - rows + 1),
                    rows=rows, dim=_log_uniform(rng, 64, 2048), params=params,
                    out=params if rng.random() < 0.7 else "bfloat16", scale=rng.choice([1.0, 45.25, 0.125]),
                    ids=rng.choice(["uniform", "skewed", "padded"]))
    if kind == "norm":
        rows = _log_uniform(rng, 1, 65536)
        stream = rng.choice(["bfloat16", "bfloat16", "float32"])
        post, gated = rng.random() < 0.6, rng.random() < 0.6
        return dict(kind=kind, train=rng.random() < 0.75, rows=rows, dim=_log_uniform(rng, 64, 4096), post=post,
                    gate=rng.choice([1, 1, _log_uniform(rng, 1, rows), rows]) if gated else 0,
                    pre=rng.random() < 0.8, block=stream if rng.random() < 0.5 else "bfloat16", stream=stream, params=params,
                    scale=rng.choice([1.0, 0.5]))
    return dict(kind=kind, layers=rng.randint(1, 4), inner=_log_uniform(rng, 64, 2048), outer=_log_uniform(rng, 8, 6144),
                vocab=rng.choice([0, _log_uniform(rng, 257, 65536)]), params=params, norm=rng.choice([2.0, 2.0, math.inf]))


# ------------------------------------------------------------------------------------ inputs
def _normal(g, shape, std, dtype):
    """Normal values on the GPU, filled in float32 and rounded once."""
    return torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(0.0, std, generator=g).to(dtype)


def _token_ids(g, case):
    """Ids over the whole vocabulary: uniform, skewed as text is (a token's rank is log-uniform, the
    frequent ones spread over the table), or sequences of skewed ids padded with id 0 at their ends."""
    n, vocab = case["tokens"], case["vocab"]
    if case["ids"] == "uniform":
        return torch.randint(0, vocab, (n,), generator=g, device=DEVICE)
    rank = torch.rand(n, generator=g, device=DEVICE, dtype=torch.float64)
    ids = ((float(vocab) ** rank).long() - 1).clamp_(0, vocab - 1)
    ids = (ids * 7919 + 11) % vocab
    if case["ids"] == "padded":
        length = max(1, n // 8)  # of every sequence, two thirds of it filled on average
        place = torch.arange(n, device=DEVICE)
        filled = torch.rand(n // length + 1, generator=g, device=DEVICE)[place // length] * 0.66 + 0.33
        ids = torch.where((place % length).float() < filled * length, ids, torch.zeros_like(ids))
    return ids


def _gradient_shapes(case):
    inner, outer, vocab = case["inner"], case["outer"], case["vocab"]
    layer = [(inner, inner), (inner // 2, inner), (inner // 2, inner), (inner, inner), (outer, inner), (inner, outer),
             (outer, inner), (inner,), (inner,), (128,), (128,)]
    return layer * case["layers"] + ([(vocab, inner), (vocab, inner), (inner,)] if vocab else [])


def _groups(case):
    """Rows of the gate: as many as asked for where they divide the rows, else the nearest below that do."""
    groups = case["gate"]
    while groups > 1 and case["rows"] % groups:
        groups -= 1
    return groups


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    params = getattr(torch, case["params"])
    if case["kind"] == "embedding":
        out = getattr(torch, case["out"])
        weight = _normal(g, (case["rows"], case["dim"]), 0.02, params).requires_grad_(case["train"])
        ids = _token_ids(g, case)
        dout = _normal(g, (case["tokens"], case["dim"]), 1e-3, out) if case["train"] else None
        padding = 0 if case["ids"] == "padded" else None
        return dict(case=case, weight=weight, ids=ids, dout=dout, padding=padding, out=out)
    if case["kind"] == "norm":
        rows, dim, train = case["rows"], case["dim"], case["train"]
        block, stream = getattr(torch, case["block"]), getattr(torch, case["stream"])
        groups = _groups(case)
        leaf = lambda t: t.requires_grad_(train)
        vector = lambda: leaf((1.0 + _normal(g, (dim,), 0.1, torch.float32)).to(params))
        # (a gate shared by all rows is a vector, one of every sequence or row a matrix [groups, 1, dim])
        gate = None
        if groups:
            gate = leaf((0.5 + _normal(g, (dim,) if groups == 1 else (groups, 1, dim), 0.2, torch.float32)).to(params))
        shape = (rows, dim) if groups <= 1 else (groups, rows // groups, dim)
        state = dict(case=case, h=leaf(_normal(g, shape, 1.5, block)), residual=leaf(_normal(g, shape, 2.0, stream)),
                     post=vector() if case["post"] else None, gate=gate, pre=vector() if case["pre"] else None, eps=1e-5)
        if train:
            state["dstream"] = _normal(g, shape, 1e-3, stream)
            state["dnormed"] = _normal(g, shape, 1e-3, block) if case["pre"] else None
        return state
    std = 10.0 ** (-2 - 2 * torch.rand(1, generator=g, device=DEVICE).item())
    parameters = []
    for shape in _gradient_shapes(case):
        p = torch.nn.Parameter(torch.empty(shape, dtype=params, device=DEVICE))
        p.grad = _normal(g, shape, std, params)
        parameters.append(p)
    # A pass clips its gradients in place.  The limit falls by a ten thousandth from pass to pass, so that
    # one on gradients that are clipped already has them all to scale again.
    limit = 0.3 * std * (math.sqrt(sum(p.numel() for p in parameters)) if case["norm"] == 2.0 else 1.0)
    return dict(case=case, parameters=parameters, limit=limit)


# ------------------------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if kind == "embedding":
        return _run_embedding(state)
    if kind == "norm":
        return _run_norm(state)
    return _run_clip(state)


def _run_embedding(state):
    case, weight, ids = state["case"], state["weight"], state["ids"]
    if own:
        from torchtitan_amd.modules.embedding import scaled_embedding

        out = scaled_embedding(ids, weight, case["scale"], padding_idx=state["padding"], first_row=case["first"],
                               dtype=state["out"])
        if not case["train"]:
            return out
        (grad,) = torch.autograd.grad(out, weight, state["dout"])
        return dict(out=out.detach(), grad=grad)
    with torch.no_grad():
        row = ids - case["first"]
        inside = (row >= 0) & (row < case["rows"])
        row = torch.where(inside, row, 0)
        values = weight[row].float() * case["scale"]
        out = torch.where(inside[:, None], values, 0.0).to(state["out"])
        if not case["train"]:
            return out
        counted = inside if state["padding"] is None else inside & (ids != state["padding"])
        parts = torch.where(counted[:, None], state["dout"].float(), 0.0)
        grad = torch.zeros(weight.shape, dtype=torch.float32, device=DEVICE).index_add_(0, row, parts)
        return dict(out=out, grad=(grad * case["scale"]).to(weight.dtype))


def _plain_norm(x, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)


def _run_norm(state):
    case, h, residual, post, gate, pre = (state[k] for k in ("case", "h", "residual", "post", "gate", "pre"))
    eps, scale = state["eps"], case["scale"]
    with torch.set_grad_enabled(case["train"]):
        if own:
            from torchtitan_amd.modules.norm import residual_rms_norm

            stream, normed = residual_rms_norm(h, residual, post_weight=post, gate=gate, pre_weight=pre,
                                               residual_scale=scale, eps=eps)
        else:
            n = h.float()
            if post is not None:
                n = _plain_norm(n, eps) * post.float()
            if gate is not None:
                n = n * gate.float()
            total = residual.float() * scale + n
            stream, normed = total.to(residual.dtype), None
            if pre is not None:
                normed = (_plain_norm(total, eps) * pre.float()).to(h.dtype)
    outputs = dict(stream=stream.detach())
    if normed is not None:
        outputs["normed"] = normed.detach()
    if case["train"]:
        results, into = [stream], [state["dstream"]]
        if normed is not None:
            results, into = results + [normed], into + [state["dnormed"]]
        leaves = [t for t in (h, residual, post, gate, pre) if t is not None]
        outputs["grads"] = torch.autograd.grad(results, leaves, into)
    return outputs


def _run_clip(state):
    parameters, kind = state["parameters"], state["case"]["norm"]
    limit = state["limit"]
    state["limit"] = limit * 0.9999
    if own:
        from torchtitan_amd.gradients import clip_grad_norm_

        total = clip_grad_norm_(parameters, limit, norm_type=kind)
        return dict(norm=total, grads=[p.grad for p in parameters])
    with torch.no_grad():
        grads = [p.grad for p in parameters]
        if kind == 2.0:
            total = torch.stack([t.float().square().sum(dtype=torch.float64) for t in grads]).sum().sqrt().float()
        else:
            total = torch.stack([t.float().abs().amax() for t in grads]).amax()
        factor = (limit / (total + 1e-6)).clamp(max=1.0)
        return dict(norm=total, grads=[t.copy_(t.float() * factor) for t in grads])


# ------------------------------------------------------------------------------------ accounts
def _expected_rows(case):
    """Rows of the table that the ids are expected to read."""
    n, vocab, share = case["tokens"], case["vocab"], case["rows"] / case["vocab"]
    if case["ids"] == "uniform":
        return share * vocab * (1.0 - (1.0 - 1.0 / vocab) ** n)
    if case["ids"] == "padded":
        n = 0.66 * n
    first = torch.arange(1, vocab + 1, dtype=torch.float64)
    chance = torch.log1p(1.0 / first) / math.log(vocab + 1.0)
    return share * float((1.0 - (1.0 - chance) ** n).sum())


def work(case):
    """Inputs once, outputs once."""
    size = lambda name: 4.0 if name == "float32" else 2.0
    if case["kind"] == "embedding":
        n, d = case["tokens"], case["dim"]
        inside = case["rows"] / case["vocab"] * n
        moved = 8.0 * n + _expected_rows(case) * d * size(case["params"]) + n * d * size(case["out"])
        flops = inside * d
        if case["train"]:
            counted = inside * (0.66 if case["ids"] == "padded" else 1.0)
            moved += counted * d * size(case["out"]) + case["rows"] * d * size(case["params"])
            flops += counted * d
        return {"bytes": moved, "flops": flops}
    if case["kind"] == "norm":
        n, vectors = float(case["rows"] * case["dim"]), case["post"] + case["pre"] + _groups(case)
        tensors = size(case["block"]) + 2 * size(case["stream"]) + (size(case["block"]) if case["pre"] else 0.0)
        flops = n * (2 + 4 * case["post"] + 2 * bool(case["gate"]) + 4 * case["pre"])
        times = 2 if case["train"] else 1  # backward: a gradient for every tensor
        return {"bytes": times * (n * tensors + vectors * case["dim"] * size(case["params"])), "flops": flops * (3 if case["train"] else 1)}
    n = float(sum(math.prod(s) for s in _gradient_shapes(case)))
    return {"bytes": 2 * n * size(case["params"]), "flops": 3 * n}


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "embedding":
            return _exact_embedding(state)
        if case["kind"] == "norm":
            return _exact_norm(state)
        return _exact_clip(state)


def _exact_embedding(state):
    case, ids = state["case"], state["ids"].tolist()
    table = torch.cat([state["weight"].detach().double() * case["scale"], torch.zeros((1, case["dim"]), dtype=torch.float64, device=DEVICE)])
    place = torch.tensor([i - case["first"] if 0 <= i - case["first"] < case["rows"] else case["rows"] for i in ids], device=DEVICE)
    out = table.index_select(0, place)
    if not case["train"]:
        return out
    if state["padding"] is not None:
        place = place.masked_fill(state["ids"] == state["padding"], case["rows"])
    # sums of equal ids as differences of running sums would lose digits: one scatter of float64 values
    table.zero_()
    table.scatter_add_(0, place[:, None].expand(-1, case["dim"]), state["dout"].double())
    return dict(out=out, grad=table[:-1] * case["scale"])


def _exact_norm(state):
    """Outputs and gradients from their formulas, written out."""
    case, eps, a = state["case"], state["eps"], state["case"]["scale"]
    h, r = state["h"].detach().double(), state["residual"].detach().double()
    post, gate, pre = (None if state[k] is None else state[k].detach().double() for k in ("post", "gate", "pre"))
    width = h.shape[-1]
    s1 = 1.0 / torch.sqrt((h * h).sum(-1, keepdim=True) / width + eps)
    n = h if post is None else h * s1 * post
    stream = a * r + (n if gate is None else gate * n)
    s2 = 1.0 / torch.sqrt((stream * stream).sum(-1, keepdim=True) / width + eps)
    outputs = dict(stream=stream)
    if pre is not None:
        outputs["normed"] = stream * s2 * pre
    if not case["train"]:
        return outputs
    over_rows = lambda t: t.reshape(-1, width).sum(0)
    d, tail = state["dstream"].double(), []
    if pre is not None:
        hat, dy = stream * s2, state["dnormed"].double()
        tail = [over_rows(dy * hat)]
        dy = dy * pre
        d = d + s2 * (dy - hat * ((dy * hat).sum(-1, keepdim=True) / width))
    grads = [a * d]
    dgate = None
    if gate is not None:
        dgate = over_rows(d * n) if gate.dim() == 1 else (d * n).sum(1, keepdim=True)
        d = d * gate
    if post is not None:
        hat = h * s1
        grads.append(over_rows(d * hat))
        d = d * post
        d = s1 * (d - hat * ((d * hat).sum(-1, keepdim=True) / width))
    outputs["grads"] = [d, *grads, *([] if dgate is None else [dgate]), *tail]
    return outputs


def _exact_clip(state):
    grads, kind = [p.grad.double() for p in state["parameters"]], state["case"]["norm"]
    if kind == 2.0:
        total = math.sqrt(math.fsum(float((t * t).sum()) for t in grads))
    else:
        total = max(float(t.abs().max()) for t in grads)
    factor = min(1.0, state["limit"] / (total + 1e-6))
    return dict(norm=torch.tensor(total, dtype=torch.float64), grads=[t.mul_(factor) for t in grads])
