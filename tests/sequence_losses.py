"""The policy and preference losses token by token in 64 bits, and inputs for them."""
import math

import numpy as np
import torch

KL = {"k1": (lambda x: x, lambda x: 1.0), "k2": (lambda x: x * x / 2, lambda x: x),
      "k3": (lambda x: math.expm1(-x) + x, lambda x: -math.expm1(-x)), "k3_swapped": (lambda x: math.expm1(x) - x, lambda x: math.expm1(x))}


def places(case):
    """Flat places of the tokens that count, by sequence."""
    n = case["log_probs"].numel()
    mask = np.ones(n, dtype=bool) if case["mask"] is None else case["mask"].cpu().numpy().reshape(-1)
    if case["offsets"] is None:
        length = case["log_probs"].shape[1]
        bounds = [(s * length, (s + 1) * length) for s in range(case["log_probs"].shape[0])]
    else:
        offsets = case["offsets"].tolist()
        bounds = list(zip(offsets, offsets[1:]))
    return [[i for i in range(a, b) if mask[i]] for a, b in bounds]


def host(t):
    return None if t is None else t.detach().cpu().double().numpy().reshape(-1)


def policy64(case, clip_eps=0.2, clip_eps_high=None, kl_coef=0.0, kl="k3", entropy_coef=0.0, ratio="token", average="token"):
    """(loss, metrics, gradient, sizes): sizes are what each gradient is the sum of, for tolerances."""
    low, high = 1 - clip_eps, 1 + (clip_eps if clip_eps_high is None else clip_eps_high)
    lp, old, ref, A = (host(case[k]) for k in ("log_probs", "old", "ref", "advantages"))
    seqs = places(case)
    grad, sizes = np.zeros(len(lp)), np.zeros(len(lp))
    tokens, filled = sum(map(len, seqs)), sum(1 for s in seqs if s)
    pg = klm = ent = mean = share = 0.0
    per_token = len(A) != len(seqs)
    for s, idx in enumerate(seqs):
        if not idx:
            continue
        x = {i: 0.0 if old is None else lp[i] - old[i] for i in idx}
        if ratio == "sequence":
            m = math.fsum(x.values()) / len(idx)
            x = {i: m for i in idx}
        w = 1 / tokens if average == "token" else 1 / filled / len(idx)
        per = 1 / tokens if ratio == "token" else 1 / filled / len(idx)
        for i in idx:
            a, r = A[i] if per_token else A[s], math.exp(x[i])
            c = min(max(r, low), high)
            pg -= w * min(r * a, c * a)
            mean += per * r
            share += per * (abs(r - c) > 1e-6)
            g = -a * r if (r <= high if a >= 0 else r >= low) else 0.0
            k = 0.0
            if ref is not None:
                y = lp[i] - ref[i]
                klm += w * KL[kl][0](y)
                k = kl_coef * KL[kl][1](y)
            ent -= lp[i] / tokens
            grad[i] = w * (g + k) + entropy_coef / tokens
            sizes[i] = w * (abs(g) + abs(k)) + entropy_coef / tokens
    return pg + kl_coef * klm - entropy_coef * ent, [pg, klm, ent, mean, share], grad, sizes


def preference64(case, beta=0.1, kind="sigmoid", label_smoothing=0.0, average_log_probs=False):
    lp, ref = host(case["log_probs"]), host(case["ref"])
    seqs = places(case)
    P = len(seqs) // 2
    x = lp if ref is None else np.where(np.isfinite(lp), lp, 0) - np.where(np.isfinite(ref), ref, 0)
    h = [math.fsum(x[i] for i in idx) / (len(idx) if average_log_probs else 1) if idx else 0.0 for idx in seqs]
    grad, number, loss = np.zeros(len(lp)), sum(1 for p in range(P) if seqs[p] or seqs[P + p]), 0.0
    soft = lambda y: math.log1p(math.exp(-abs(y))) + max(-y, 0.0)
    sigma = lambda y: 1 / (1 + math.exp(-y)) if y > -700 else 0.0
    for p in range(P):
        if not seqs[p] and not seqs[P + p]:
            continue
        z = h[p] - h[P + p]
        if kind == "sigmoid":
            value = (1 - label_smoothing) * soft(beta * z) + label_smoothing * soft(-beta * z)
            d = beta * (label_smoothing * sigma(beta * z) - (1 - label_smoothing) * sigma(-beta * z))
        elif kind == "hinge":
            value, d = max(0.0, 1 - beta * z), -beta if beta * z < 1 else 0.0
        else:
            value, d = (z - 0.5 / beta) ** 2, 2 * (z - 0.5 / beta)
        loss += value / number
        for s, sign in ((p, 1), (P + p, -1)):
            for i in seqs[s]:
                grad[i] = sign * d / number / (len(seqs[s]) if average_log_probs else 1)
    return loss, [beta * v for v in h], grad


def tokens_of(shape, device, *, offsets=None, mask=None, dtype=torch.float32, old=True, ref=True, per_token=False, seed=0,
              outside=-math.inf):
    """Inputs; tokens that do not count hold `outside`."""
    g = torch.Generator().manual_seed(seed)
    lp = -torch.randn(shape, generator=g).abs() * 1.5
    values = dict(log_probs=lp, old=lp + 0.25 * torch.randn(shape, generator=g), ref=lp + 0.4 * torch.randn(shape, generator=g))
    sequences = shape[0] if offsets is None else len(offsets) - 1
    advantages = torch.randn(shape if per_token else (sequences,), generator=g)
    if sequences > 2 and not per_token:
        advantages[1] = 0.0
    offsets = None if offsets is None else torch.tensor(offsets)
    if mask is not None:
        mask = torch.rand(shape, generator=g) < mask
        if mask.dim() == 2 and mask.shape[0] > 2:
            mask[2] = False
        values = {k: torch.where(mask, v, outside) for k, v in values.items()}
        if per_token:
            advantages = torch.where(mask, advantages, math.nan)
    case = dict({k: v.to(dtype) for k, v in values.items()}, advantages=advantages, offsets=offsets, mask=mask)
    if not old:
        case["old"] = None
    if not ref:
        case["ref"] = None
    case = {k: None if t is None else t.to(device) for k, t in case.items()}
    case["log_probs"].requires_grad_(True)
    return case


def check_policy(call, case, dloss=0.5, **options):
    loss, metrics = call(case["log_probs"], case["advantages"], case["old"], case["ref"], offsets=case["offsets"], mask=case["mask"],
                         **options)
    want, want_metrics, want_grad, sizes = policy64(case, **options)
    (grad,) = torch.autograd.grad(loss, case["log_probs"], torch.tensor(dloss, device=loss.device))
    close(loss, metrics, grad, want, want_metrics, dloss * want_grad, dloss * sizes, case)


def check_preference(call, case, dloss=0.5, **options):
    loss, rewards = call(case["log_probs"], case["ref"], offsets=case["offsets"], mask=case["mask"], **options)
    want, want_rewards, want_grad = preference64(case, **options)
    (grad,) = torch.autograd.grad(loss, case["log_probs"], torch.tensor(dloss, device=loss.device))
    close(loss, rewards, grad, want, want_rewards, dloss * want_grad, np.abs(dloss * want_grad), case)


def close(loss, more, grad, want, want_more, want_grad, sizes, case):
    """Everything is formed in 64 bits (1e-12 of its parts for their order and last bits) and rounded once."""
    u = 2.0 ** -24
    size = max([1.0, abs(want), *map(abs, want_more)])
    assert loss.dtype == torch.float32 and loss.shape == () and abs(loss.item() - want) <= u * abs(want) + 1e-12 * size
    assert more.dtype == torch.float32 and more.shape == (len(want_more),) and not more.requires_grad
    assert all(abs(a - b) <= u * abs(b) + 1e-12 * size for a, b in zip(more.tolist(), want_more))
    half = torch.finfo(grad.dtype).eps / 2
    assert grad.dtype == case["log_probs"].dtype and grad.shape == case["log_probs"].shape
    got = grad.cpu().double().numpy().reshape(-1)
    assert np.all(np.abs(got - want_grad) <= half * np.abs(want_grad) + 1e-11 * sizes + 1e-40)
    assert np.all(got[sizes == 0] == 0)
