"""The two ends of a policy or preference training step, as a user's program calls them.

The clipped policy loss with its KL term and the preference loss of paired sequences, each with its
gradient, from the log-probabilities of packed or padded sequences; and the AdamW step over a list of
parameters, with moments in 32 bits or in 8.  Sizes are those of the benchmark, the tests and the layer
shapes they name (147 456 packed tokens of 16 sequences, model size 2048 with hidden size 6144,
vocabulary 151 936, the tests' 128 x 512 layer) and of counts around them, packed, padded and ragged.

``listed()`` gives the fixed cases, ``draw(rng)`` another one of the same ranges, ``prepare`` what a
program holds before the call, ``run`` one pass -- with ``own`` through the framework's operators, else
in elementary torch operations --, ``work`` the bytes and operations a pass cannot do without, ``exact``
the results in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # A trainer's micro-batch of short completions, padded to the longest, one of them masked out whole:
        # token ratios, KL against the reference policy.  The smallest call, where latency counts.
        dict(name="policy_padded_short", kind="policy", layout="padded", sequences=16, tokens=16 * 61, behind=0, values="float32",
             ratio="token", average="token", kl="k3", kl_coef=0.05, entropy_coef=0.0, low=0.2, high=0.28, old=True, ref=True,
             advantage="sequence", train=True),
        # All packed tokens of one policy step, one ratio a sequence, KL and entropy terms.
        dict(name="policy_packed_sequence_ratio", kind="policy", layout="packed", sequences=16, tokens=147456, behind=0,
             values="float32", ratio="sequence", average="sequence", kl="k3_swapped", kl_coef=0.1, entropy_coef=0.01, low=0.2,
             high=0.2, old=True, ref=True, advantage="sequence", train=True),
        # A rollout batch of 1024 sequences of up to 4099 tokens, padded, an advantage for every token.
        dict(name="policy_padded_rollout", kind="policy", layout="padded", sequences=1024, tokens=1024 * 4099, behind=0,
             values="float32", ratio="token", average="token", kl="k3", kl_coef=0.02, entropy_coef=0.001, low=0.2, high=0.2,
             old=True, ref=True, advantage="token", train=True),
        # Eight pairs of a preference set, prompts masked out.  The smallest preference loss.
        dict(name="preference_few_pairs", kind="preference", layout="padded", sequences=16, tokens=16 * 509, behind=0,
             values="float32", loss="sigmoid", beta=0.1, smoothing=0.0, mean=False, ref=True, train=True),
        # 512 pairs of long answers, packed, mean log-ratios and the squared loss.
        dict(name="preference_packed_pairs", kind="preference", layout="packed", sequences=1024, tokens=2097152, behind=77,
             values="bfloat16", loss="ipo", beta=0.1, smoothing=0.0, mean=True, ref=True, train=True),
        # One layer of a model as small as the tests': nine small tensors.  The smallest update.
        dict(name="adamw_small_layer", kind="adamw", bits=32, inner=128, outer=512, experts=0, vocab=0, params="bfloat16",
             master=False, clip=False, decay=0.1),
        # One layer in bf16 with float32 master weights, gradients clipped as they are read.
        dict(name="adamw_layer_master", kind="adamw", bits=32, inner=2048, outer=6144, experts=0, vocab=0, params="bfloat16",
             master=True, clip=True, decay=0.1),
        # A layer with embedding and head in float32: 673 million parameters.
        dict(name="adamw_model_float32", kind="adamw", bits=32, inner=2048, outer=6144, experts=0, vocab=151936, params="float32",
             master=False, clip=True, decay=0.01),
        # The same three with moments in 8 bits: the small layer,
        dict(name="adamw8_small_layer", kind="adamw", bits=8, inner=128, outer=512, experts=0, vocab=0, params="float32",
             master=False, clip=False, decay=0.0),
        # one layer,
        dict(name="adamw8_layer", kind="adamw", bits=8, inner=2048, outer=6144, experts=0, vocab=0, params="bfloat16", master=True,
             clip=True, decay=0.1),
        # and the model, with 128 experts of hidden size 768, in bf16: 1277 million parameters.
        dict(name="adamw8_model", kind="adamw", bits=8, inner=2048, outer=6144, experts=128, vocab=151936, params="bfloat16",
             master=False, clip=False, decay=0.1),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["policy", "policy", "preference", "adamw", "adamw"])
    if kind == "adamw":
        params = rng.choice(["bfloat16", "bfloat16", "float32"])
        return dict(kind=kind, bits=rng.choice([32, 8]), inner=_log_uniform(rng, 33, 2048), outer=_log_uniform(rng, 8, 6144),
                    experts=rng.choice([0, 0, _log_uniform(rng, 1, 32)]), vocab=rng.choice([0, _log_uniform(rng, 257, 65536)]),
                    params=params, master=params == "bfloat16" and rng.random() < 0.5, clip=rng.random() < 0.5, decay=rng.choice([0.0, 0.1]))
    sequences = 2 * _log_uniform(rng, 1, 512)
    length = _log_uniform(rng, 1, 4096)
    layout = rng.choice(["packed", "padded"])
    tokens = sequences * length - (rng.randrange(length) if layout == "packed" else 0)
    shared = dict(kind=kind, layout=layout, sequences=sequences, tokens=tokens,
                  behind=rng.choice([0, min(tokens, rng.randint(1, 300))]) if layout == "packed" else 0,
                  values=rng.choice(["float32", "float32", "bfloat16"]), train=rng.random() < 0.8, ref=rng.random() < 0.8)
    if kind == "preference":
        loss = rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"])
        return dict(shared, loss=loss, beta=rng.choice([0.05, 0.1, 0.5]), mean=rng.random() < 0.4,
                    smoothing=rng.choice([0.0, 0.1]) if loss == "sigmoid" else 0.0)
    ratio = rng.choice(["token", "token", "sequence"])
    return dict(shared, ratio=ratio, average=rng.choice(["token", "sequence"]), kl=rng.choice(["k1", "k2", "k3", "k3_swapped"]),
                kl_coef=rng.choice([0.01, 0.1]) if shared["ref"] else 0.0, entropy_coef=rng.choice([0.0, 0.01]),
                low=rng.choice([0.1, 0.2]), high=rng.choice([0.2, 0.28]), old=rng.random() < 0.8,
                advantage="sequence" if ratio == "sequence" else rng.choice(["sequence", "token"]))


# ------------------------------------------------------------------------------------ inputs
def _normal(g, shape, std, dtype):
    """Normal values on the GPU, filled in float32 and rounded once."""
    return torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(0.0, std, generator=g).to(dtype)


def _shapes(case):
    """Four attention projections, three of a feed-forward block and two norms; stacks of experts; embedding and head."""
    inner, outer, vocab, experts = case["inner"], case["outer"], case["vocab"], case["experts"]
    shapes = [(inner, inner), (inner // 2, inner), (inner // 2, inner), (inner, inner), (outer, inner), (inner, outer),
              (outer, inner), (inner,), (128,)]
    if experts:
        shapes += [(experts, 768, inner), (experts, inner, 768), (experts, 768, inner)]
    return shapes + ([(vocab, inner), (vocab, inner)] if vocab else [])


def _prepare_sequences(case, g):
    """Log-probabilities of sampled tokens, and which of them count: sequences in a row between `offsets`, of any length
    from none on; or one row a sequence with a mask -- its prompt, the padding behind its end and one sequence
    out of eight or so are out, and a masked place holds what a masked token has, minus infinity."""
    S, T, values = case["sequences"], case["tokens"], getattr(torch, case["values"])
    packed = case["layout"] == "packed"
    shape = (T,) if packed else (S, T // S)
    state = dict(case=case, offsets=None, mask=None)
    policy = -_normal(g, shape, 1.5, torch.float32).abs() - 1e-3
    old = policy + _normal(g, shape, 0.15, torch.float32)
    ref = policy + _normal(g, shape, 0.3, torch.float32)
    if packed:
        cuts = torch.randint(0, T - case["behind"] + 1, (S - 1,), generator=g, device=DEVICE).sort().values
        ends = torch.tensor([0, T - case["behind"]], device=DEVICE)
        state["offsets"] = torch.cat((ends[:1], cuts, ends[1:]))
    else:
        length = T // S
        place = torch.arange(length, device=DEVICE)
        filled = torch.rand(S, 1, generator=g, device=DEVICE)
        begin, end = (filled * 0.3 * length).long(), ((0.4 + 0.6 * filled) * length).long().clamp(min=1)
        out = torch.rand(S, 1, generator=g, device=DEVICE) < 0.12
        state["mask"] = (place >= begin) & (place < end) & ~out
        nothing = torch.where(state["mask"], 0.0, -math.inf)
        policy, old, ref = policy + nothing, old + nothing, ref + nothing
    state["log_probs"] = policy.to(values).requires_grad_(case["train"])
    state["ref"] = ref.to(values) if case["ref"] else None
    if case["kind"] == "policy":
        state["old"] = old.to(values) if case["old"] else None
        state["advantages"] = _normal(g, (S,) if case["advantage"] == "sequence" else shape, 1.0, torch.float32)
    # (of four micro-batches whose gradients are added up)
    state["dloss"] = torch.full((), 0.25, device=DEVICE)
    return state


BLOCK = 32  # values of a moment in 8 bits that share a scale
# The two forms of 8 bits, as (exponent bias, float32 bits below a code's last, largest code, exponent of the largest): the
# first moment has a sign, 4 bits of exponent and 3 of mantissa, the second 5 bits of exponent and 3 of mantissa.
FIRST, SECOND = (7, 20, 126, 8), (15, 20, 255, 16)


def _mixed(x):
    """32 bits that each depend on all bits of the 32-bit numbers `x`, held in int64."""
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _dither(n, seed, step, number):
    """The 16 random bits of each of n values, from the optimizer's seed, the step and the parameter's number."""
    key = 0
    for word in (seed & 0xFFFFFFFF, seed >> 32, step, number):
        key = _mixed((key + word + 0x9E3779B9) & 0xFFFFFFFF)
    pair = torch.arange(-(-n // 2), dtype=torch.int64, device=DEVICE)
    bits = _mixed((pair * 0x9E3779B9 + key) & 0xFFFFFFFF)
    return torch.stack((bits & 0xFFFF, bits >> 16), 1).reshape(-1)[:n]


def _in_blocks(x):
    """A parameter's values as whole blocks, zeros behind the last."""
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _encode(x, form, dither):
    """(codes, scales) of float32 blocks; a value between two codes becomes the upper one with the probability of its
    distance from the lower."""
    bias, shift, largest, top = form
    bits = x.abs().view(torch.int32).long()
    amax = bits.amax(1)
    ceiling = 0x1FFFFF if form is FIRST else 0x0FFFFF
    scale = torch.where(amax > 0, ((amax + ceiling) >> 23) - top, 0).clamp(0, 254)
    scale = torch.where(amax >= 0x7F800000, 255, scale)
    at = torch.ldexp(x.abs().double(), (bias - scale).double()[:, None]).float()  # a code in the topmost bits
    code = (at.view(torch.int32).long() + (dither.view(-1, BLOCK) << (shift - 16)) + (1 << (shift - 17))) >> shift
    code = torch.where(x == 0, 0, code.clamp(max=largest))
    code = torch.where(scale[:, None] == 255, largest, code)
    if form is SECOND:
        code = torch.where(x > 0, code.clamp(min=1), code)
    else:
        code = code | (x.signbit().long() << 7)
    return code.to(torch.uint8), scale.to(torch.uint8)


def _decode(codes, scales, form):
    """float32 values of codes [blocks, 32]."""
    bias, shift, _, _ = form
    code, scale = codes.long(), scales.long()
    size = (code & 127 if form is FIRST else code).to(torch.int32) << shift
    value = torch.ldexp(size.view(torch.float32).double(), (scale - bias).double()[:, None]).float()
    value = torch.where(scale[:, None] == 255, math.nan, value)
    return torch.where(code >= 128, -value, value) if form is FIRST else value


def _prepare_adamw(case, g, seed):
    params = getattr(torch, case["params"])
    std = 10.0 ** (-2 - 2 * torch.rand(1, generator=g, device=DEVICE).item())
    state = dict(case=case, parameters=[], moments=[], masters=[], step=100, seed=seed * 7919 + 3, number=0)
    for shape in _shapes(case):
        weight = _normal(g, shape, 0.02, torch.float32)
        p = torch.nn.Parameter(weight.to(params))
        p.grad = _normal(g, shape, std, params)
        first = _normal(g, shape, 0.3 * std, torch.float32)
        second = _normal(g, shape, std, torch.float32).square_()
        if case["bits"] == 8:
            nothing = torch.full((_in_blocks(first).numel(),), 1 << 15, dtype=torch.int64, device=DEVICE)
            state["moments"].append(_encode(_in_blocks(first), FIRST, nothing) + _encode(_in_blocks(second), SECOND, nothing))
        else:
            state["moments"].append((first, second))
        state["masters"].append(weight if case["master"] else None)
        state["parameters"].append(p)
    count = sum(p.numel() for p in state["parameters"])
    # (clipped to a third of the norm that such gradients have)
    state["norm"] = torch.full((), std * math.sqrt(count), device=DEVICE) if case["clip"] else None
    state["limit"] = std * math.sqrt(count) / 3
    return state


HYPER = dict(lr=3e-4, betas=(0.9, 0.95), eps=1e-8)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "adamw":
        return _prepare_adamw(case, g, seed)
    return _prepare_sequences(case, g)


# ------------------------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if kind == "adamw":
        return _run_adamw(state)
    return _run_policy(state) if kind == "policy" else _run_preference(state)


def _result(state, loss, more, grad):
    return dict(more, loss=loss, grad=grad) if state["case"]["train"] else dict(more, loss=loss)


def _counted(state):
    """(sequence of every token, whether it counts), flat."""
    log_probs, S = state["log_probs"], state["case"]["sequences"]
    place = torch.arange(log_probs.numel(), device=DEVICE)
    if state["offsets"] is None:
        sequence = place // (log_probs.numel() // S)
        inside = torch.ones_like(place, dtype=torch.bool)
    else:
        sequence = torch.bucketize(place, state["offsets"][1:], right=True).clamp(max=S - 1)
        inside = (place >= state["offsets"][0]) & (place < state["offsets"][-1])
    return sequence, inside if state["mask"] is None else inside & state["mask"].reshape(-1)


def _sums(sequence, values, S):
    """Sums over every sequence's tokens, in 64 bits."""
    return torch.zeros(S, dtype=torch.float64, device=DEVICE).index_add_(0, sequence, values.double())


def _kl(x, kind):
    """The estimator of the KL term at a log-ratio x of policy and reference, and its derivative."""
    if kind == "k1":
        return x, torch.ones_like(x)
    if kind == "k2":
        return x * x * 0.5, x
    if kind == "k3":
        return torch.expm1(-x) + x, -torch.expm1(-x)
    return torch.expm1(x) - x, torch.expm1(x)


def _run_policy(state):
    case, log_probs = state["case"], state["log_probs"]
    if own:
        from torchtitan_amd.rl import policy_loss

        loss, metrics = policy_loss(log_probs, state["advantages"], state["old"], state["ref"], offsets=state["offsets"],
                                    mask=state["mask"], clip_eps=case["low"], clip_eps_high=case["high"],
                                    kl_coef=case["kl_coef"], kl=case["kl"], entropy_coef=case["entropy_coef"],
                                    ratio=case["ratio"], average=case["average"], advantage=case["advantage"])
        if not case["train"]:
            return dict(metrics=metrics, loss=loss)
        (grad,) = torch.autograd.grad(loss, log_probs, state["dloss"])
        return _result(state, loss.detach(), dict(metrics=metrics), grad)
    with torch.no_grad():
        S, whole = case["sequences"], case["ratio"] == "sequence"
        sequence, counts = _counted(state)
        # (in 64 bits: which side of a clipping border a ratio is on decides about its whole gradient)
        flat = lambda t: torch.where(counts, t.reshape(-1).double(), 0.0)
        lp = flat(log_probs)
        x = lp - flat(state["old"]) if case["old"] else torch.zeros_like(lp)
        n = _sums(sequence, counts, S)
        tokens, filled = n.sum().clamp(min=1), (n > 0).sum().clamp(min=1)
        if whole:
            x = (_sums(sequence, x, S) / n.clamp(min=1))[sequence]
        A = state["advantages"].reshape(-1) if case["advantage"] == "token" else state["advantages"][sequence]
        A = torch.where(counts, A.double(), 0.0)
        ratio = torch.exp(x)
        clipped = ratio.clamp(1 - case["low"], 1 + case["high"])
        objective = -torch.minimum(ratio * A, clipped * A)
        active = torch.where(A >= 0, ratio <= 1 + case["high"], ratio >= 1 - case["low"])
        each = torch.where(counts, (1 / tokens).expand_as(counts) if case["average"] == "token" else
                           (1 / (filled * n.clamp(min=1)))[sequence], 0.0)
        kl, slope = _kl(lp - flat(state["ref"]), case["kl"]) if case["ref"] else (torch.zeros_like(lp), torch.zeros_like(lp))
        pg, kl_div, entropy = (objective * each).sum(), (kl * each).sum(), -lp.sum() / tokens
        loss = pg + case["kl_coef"] * kl_div - case["entropy_coef"] * entropy
        # (means over tokens, or over sequences where there is a ratio for each)
        per = torch.where(counts, 1 / (filled * n.clamp(min=1))[sequence] if whole else 1 / tokens, 0.0)
        ratio_mean = (ratio * per).sum()
        share = (((ratio - clipped).abs() > 1e-6) * per).sum()
        metrics = torch.stack([pg, kl_div, entropy, ratio_mean, share]).float()
        if not case["train"]:
            return dict(metrics=metrics, loss=loss.float())
        weight = torch.where(active, -A * ratio, 0.0)
        grad = weight * each + case["kl_coef"] * slope * each
        grad = grad + torch.where(counts, case["entropy_coef"] / tokens, 0.0)
        grad = (grad * state["dloss"]).to(log_probs.dtype).view(log_probs.shape)
        return _result(state, loss.float(), dict(metrics=metrics), grad)


def _run_preference(state):
    case, log_probs = state["case"], state["log_probs"]
    if own:
        from torchtitan_amd.rl import preference_loss

        loss, rewards = preference_loss(log_probs, state["ref"], offsets=state["offsets"], mask=state["mask"],
                                        beta=case["beta"], kind=case["loss"], label_smoothing=case["smoothing"],
                                        average_log_probs=case["mean"])
        if not case["train"]:
            return dict(rewards=rewards, loss=loss)
        (grad,) = torch.autograd.grad(loss, log_probs, state["dloss"])
        return _result(state, loss.detach(), dict(rewards=rewards), grad)
    with torch.no_grad():
        S, beta, smoothing = case["sequences"], case["beta"], case["smoothing"]
        sequence, counts = _counted(state)
        flat = lambda t: torch.where(counts, t.reshape(-1).float(), 0.0)
        x = flat(log_probs) - flat(state["ref"]) if case["ref"] else flat(log_probs)
        n = _sums(sequence, counts, S)
        each = 1 / n.clamp(min=1) if case["mean"] else torch.ones_like(n)
        h = _sums(sequence, x, S) * each
        z = h[:S // 2] - h[S // 2:]
        pairs = (n[:S // 2] + n[S // 2:]) > 0
        if case["loss"] == "sigmoid":
            soft = lambda y: torch.log1p(torch.exp(-y.abs())) + torch.clamp(-y, min=0)  # -log sigmoid(y)
            losses = (1 - smoothing) * soft(beta * z) + smoothing * soft(-beta * z)
            slope = beta * (smoothing * torch.sigmoid(beta * z) - (1 - smoothing) * torch.sigmoid(-beta * z))
        elif case["loss"] == "hinge":
            losses = torch.clamp(1 - beta * z, min=0)
            slope = torch.where(beta * z < 1, -beta, 0.0)
        else:
            losses = (z - 0.5 / beta) ** 2
            slope = 2 * (z - 0.5 / beta)
        number = pairs.sum().clamp(min=1)
        loss = (torch.where(pairs, losses, 0.0).sum() / number).float()
        rewards = (beta * h).float()
        if not case["train"]:
            return dict(rewards=rewards, loss=loss)
        slope = torch.where(pairs, slope, 0.0) / number
        slope = torch.cat((slope, -slope)) * each
        grad = (torch.where(counts, slope[sequence], 0.0) * state["dloss"]).to(log_probs.dtype).view(log_probs.shape)
        return _result(state, loss, dict(rewards=rewards), grad)


def _run_adamw(state):
    case, parameters = state["case"], state["parameters"]
    if own:
        if "optimizer" not in state:  # (made once, and then kept, as a program does)
            from torchtitan_amd.optimizers import AdamW

            state["optimizer"] = AdamW(parameters, **HYPER, weight_decay=case["decay"], state_bits=case["bits"],
                                       master_weights=case["master"], seed=state["seed"])
            names = ("exp_avg", "exp_avg_sq") if case["bits"] == 32 else ("exp_avg", "exp_avg_scale", "exp_avg_sq",
                                                                          "exp_avg_sq_scale")
            for p, moments, master in zip(parameters, state["moments"], state["masters"]):
                state["optimizer"].state[p] = dict(zip(names, moments), step=state["step"])
                if master is not None:
                    state["optimizer"].state[p]["master"] = master
        optimizer = state["optimizer"]
        if case["clip"]:
            optimizer.step(total_norm=state["norm"], max_norm=state["limit"])
        else:
            optimizer.step()
        moments = optimizer.moments() if case["bits"] == 8 else state["moments"]
    else:
        state["step"] += 1
        moments = [_update(state, i) for i in range(len(parameters))]
    out = dict(parameters=[p.detach() for p in parameters], first=[m[0] for m in moments], second=[m[1] for m in moments])
    return dict(out, masters=state["masters"]) if case["master"] else out


@torch.no_grad()
def _update(state, i):
    """One parameter's update in place; its moments as values."""
    case, p, step = state["case"], state["parameters"][i], state["step"]
    (b1, b2), lr, eps = HYPER["betas"], HYPER["lr"], HYPER["eps"]
    g = p.grad.float()
    if case["clip"]:
        g = g * torch.clamp(state["limit"] / (state["norm"] + 1e-6), max=1.0)
    if case["bits"] == 8:
        n, shape = p.numel(), p.shape
        c1, s1, c2, s2 = state["moments"][i]
        m, v = (_decode(c, s, f).reshape(-1)[:n].view(shape) for c, s, f in ((c1, s1, FIRST), (c2, s2, SECOND)))
    else:
        m, v = state["moments"][i]
    m_new = m * b1 + g * (1 - b1)
    v_new = v * b2 + g * g * (1 - b2)
    w = state["masters"][i] if case["master"] else p
    root = torch.sqrt(v_new) * (1 / math.sqrt(1 - b2 ** step)) + eps
    new = w.float() * (1 - lr * case["decay"]) - (lr / (1 - b1 ** step)) * (m_new / root)
    w.copy_(new)
    if case["master"]:
        p.copy_(new)
    if case["bits"] == 32:
        m.copy_(m_new)
        v.copy_(v_new)
        return m, v
    dither = _dither(n, state["seed"], step, i)
    dither = torch.nn.functional.pad(dither, (0, -n % BLOCK))
    values = []
    for x, c, s, f in ((m_new, c1, s1, FIRST), (v_new, c2, s2, SECOND)):
        codes, scales = _encode(_in_blocks(x), f, dither)
        c.copy_(codes)
        s.copy_(scales)
        values.append(_decode(codes, scales, f).reshape(-1)[:n].view(shape).to(torch.bfloat16))
    return tuple(values)


# ------------------------------------------------------------------------------------ cost
def work(case):
    size = {"bfloat16": 2, "float32": 4}
    if case["kind"] != "adamw":
        T, S = case["tokens"], case["sequences"]
        arrays = 1 + case["ref"] + case.get("old", False) + case["train"]
        moved = arrays * size[case["values"]] * T + (T if case["layout"] == "padded" else 8 * (S + 1))
        if case["kind"] == "policy":
            moved += 4 * (T if case["advantage"] == "token" else S)
        else:
            moved += 4 * S
        return {"bytes": moved, "flops": 20 * T}
    n, p = sum(math.prod(s) for s in _shapes(case)), size[case["params"]]
    # the gradient is read, the parameter written, it or its master weight read, the master written
    moved = 2 * p + (8 if case["master"] else p)
    # moments read and written; in 8 bits with a scale for every 32, and their values written
    moved += 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4
    return {"bytes": int(n * moved), "flops": 15 * n}


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "adamw":
        return _exact_adamw(state)
    log_probs = state["log_probs"].detach()
    host = lambda t: None if t is None else t.cpu().double().numpy()
    lp, ref, old, A = (host(t) for t in (log_probs, state["ref"], state.get("old"), state.get("advantages")))
    S, T = case["sequences"], case["tokens"]
    if case["layout"] == "padded":
        length = T // S
        bounds = [(s * length, (s + 1) * length) for s in range(S)]
        mask = state["mask"].cpu().numpy().reshape(-1)
    else:
        offsets = state["offsets"].tolist()
        bounds = list(zip(offsets, offsets[1:]))
        mask = np.ones(T, dtype=bool)
    lp, ref, old = (None if t is None else t.reshape(-1) for t in (lp, ref, old))
    places = [np.arange(a, b)[mask[a:b]] for a, b in bounds]
    grad = np.zeros(T)
    result = (_exact_policy if case["kind"] == "policy" else _exact_preference)(case, lp, ref, old, A, places, grad)
    if case["train"]:
        result["grad"] = 0.25 * grad.reshape(log_probs.shape)
    return {k: torch.as_tensor(np.asarray(v, dtype=np.float64)) for k, v in result.items()}


def _exact_policy(case, lp, ref, old, A, places, grad):
    tokens, filled = sum(len(i) for i in places), sum(len(i) > 0 for i in places)
    pg = kl_div = entropy = mean = share = 0.0
    for s, i in enumerate(places):
        if not len(i):
            continue
        x = lp[i] - old[i] if old is not None else np.zeros(len(i))
        if case["ratio"] == "sequence":
            x = np.full(len(i), x.mean())
        a = A.reshape(-1)[i] if case["advantage"] == "token" else np.full(len(i), A[s])
        r, low, high = np.exp(x), 1 - case["low"], 1 + case["high"]
        # the smaller of the two objectives, by the sign of the advantage
        inside = np.where(a >= 0, r <= high, r >= low)
        each = 1 / tokens if case["average"] == "token" else 1 / (filled * len(i))
        pg -= (a * np.where(a >= 0, np.minimum(r, high), np.maximum(r, low))).sum() * each
        grad[i] = np.where(inside, -a * r, 0.0) * each
        if ref is not None:
            y = lp[i] - ref[i]
            kl, slope = {"k1": lambda: (y, np.ones_like(y)), "k2": lambda: (y * y / 2, y),
                         "k3": lambda: (np.expm1(-y) + y, -np.expm1(-y)),
                         "k3_swapped": lambda: (np.expm1(y) - y, np.expm1(y))}[case["kl"]]()
            kl_div += kl.sum() * each
            grad[i] += case["kl_coef"] * slope * each
        entropy -= lp[i].sum() / tokens
        grad[i] += case["entropy_coef"] / tokens
        per = 1 / tokens if case["ratio"] == "token" else 1 / (filled * len(i))
        mean += r.sum() * per
        share += (np.abs(r - np.clip(r, low, high)) > 1e-6).sum() * per
    loss = pg + case["kl_coef"] * kl_div - case["entropy_coef"] * entropy
    return dict(metrics=[pg, kl_div, entropy, mean, share], loss=loss)


def _exact_preference(case, lp, ref, old, A, places, grad):
    pairs, beta, e = len(places) // 2, case["beta"], case["smoothing"]
    h = np.zeros(2 * pairs)
    for s, i in enumerate(places):
        if len(i):
            x = lp[i] - (ref[i] if ref is not None else 0.0)
            h[s] = x.mean() if case["mean"] else x.sum()
    counted = [k for k in range(pairs) if len(places[k]) + len(places[pairs + k])]
    loss = 0.0
    for k in counted:
        z = h[k] - h[pairs + k]
        if case["loss"] == "sigmoid":
            value = (1 - e) * np.logaddexp(0, -beta * z) + e * np.logaddexp(0, beta * z)
            slope = beta * (1 / (1 + np.exp(-beta * z)) - (1 - e))
        elif case["loss"] == "hinge":
            value, slope = max(0.0, 1 - beta * z), -beta if beta * z < 1 else 0.0
        else:
            value, slope = (z - 1 / (2 * beta)) ** 2, 2 * (z - 1 / (2 * beta))
        loss += value / len(counted)
        for s, sign in ((k, 1), (pairs + k, -1)):
            i = places[s]
            if len(i):
                grad[i] = sign * slope / len(counted) / (len(i) if case["mean"] else 1)
    return dict(rewards=beta * h, loss=loss)


def _exact_rounded(x, form, dither):
    """The values that 64-bit blocks are held as in 8 bits."""
    largest, (bias, _, _, top) = (448.0, form) if form is FIRST else (122880.0, form)
    amax = x.abs().amax(1, keepdim=True)
    scale = torch.ceil(torch.log2((amax / largest).clamp(min=2.0 ** -127))).clamp(-127, 127)
    y = x.abs() * torch.exp2(-scale)
    unit = torch.exp2(torch.floor(torch.log2(y.clamp(min=1e-300))).clamp(min=1 - bias) - 3)
    y = torch.floor(y / unit + (dither.view(-1, BLOCK) + 0.5) / 65536) * unit
    if form is SECOND:
        y = torch.where((x > 0) & (y == 0), unit, y)
    return torch.sign(x) * torch.clamp(y, max=largest) * torch.exp2(scale)


@torch.no_grad()
def _exact_adamw(state):
    case, step = state["case"], state["step"] + 1
    (b1, b2), lr, eps = HYPER["betas"], HYPER["lr"], HYPER["eps"]
    out = dict(parameters=[], first=[], second=[])
    if case["master"]:
        out["masters"] = []
    for i, p in enumerate(state["parameters"]):
        g = p.grad.double()
        if case["clip"]:
            norm = state["norm"].double()
            g = g * torch.clamp(state["limit"] / (norm + 1e-6), max=1.0)
        moments, n = state["moments"][i], p.numel()
        if case["bits"] == 8:
            m, v = (_decode(*moments[k:k + 2], f).double().reshape(-1)[:n].view(p.shape) for k, f in ((0, FIRST), (2, SECOND)))
        else:
            m, v = (t.double() for t in moments)
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        w = (state["masters"][i] if case["master"] else p).double()
        w = w - lr * case["decay"] * w - lr * (m / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + eps)
        if case["bits"] == 8:
            dither = torch.nn.functional.pad(_dither(n, state["seed"], step, i), (0, -n % BLOCK))
            m, v = (_exact_rounded(_in_blocks(x), f, dither).reshape(-1)[:n].view(p.shape) for x, f in ((m, FIRST), (v, SECOND)))
        for name, value in (("parameters", w), ("first", m), ("second", v)):
            out[name].append(value.float() if name != "parameters" and case["bits"] == 8 else value)
        if case["master"]:
            out["masters"].append(w)
    return out
