"""GRPO / PPO policy-gradient loss with per-token KL, and the per-token log-probabilities under
it (torchtitan/experiments/rl/unified/actors/utils.py:11-147).

Same functions, arguments, return values and formulas as the reference.  The one heavy step,
log-softmax over the vocabulary in float32 followed by a gather of the generated tokens, runs
as one HIP kernel over the bf16 logits (and one more in backward) whenever the logits are a
bf16 GPU tensor; otherwise the same torch ops as the reference run.

``policy_loss`` is the loss itself over the tokens of a whole batch, packed or padded, with ratios of tokens or of sequences, and
``preference_loss`` that of pairs of sequences: two launches forward and one backward on the GPU, elsewhere the same
formula in torch operations.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from .. import _lib, ops
from ..modules.norm import _Refusing


class _TokenLogProbs(torch.autograd.Function):
    """log_softmax(logits.float(), -1).gather(1, target[:, None]).squeeze(-1) for bf16 logits."""

    @staticmethod
    def forward(ctx, logits, target):
        lp, lse = ops.token_logprob_fwd(logits, target)
        ctx.save_for_backward(logits, target, lse)
        return lp

    @staticmethod
    def backward(ctx, grad):
        logits, target, lse = ctx.saved_tensors
        return _once(ops.token_logprob_bwd(logits, target, lse, grad)), None


def token_log_probs(logits: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
    """float32 log-probability of target[r] under softmax(logits[r]); logits [rows, vocab]."""
    if logits.is_cuda and logits.dtype == torch.bfloat16 and logits.dim() == 2:
        return _TokenLogProbs.apply(logits, target)
    log_probs = F.log_softmax(logits.to(torch.float32), dim=-1)
    return log_probs.gather(1, target.unsqueeze(-1)).squeeze(-1)


def compute_token_log_probs(model: torch.nn.Module, prompt_token_ids: list[int],
                            gen_token_ids: list[int], device: torch.device) -> torch.Tensor:
    """Per-token log-probabilities of the generated tokens under `model` (one forward over
    prompt + completion; position i predicts token i + 1)."""
    full = torch.tensor(prompt_token_ids + gen_token_ids, dtype=torch.long, device=device).unsqueeze(0)
    logits = model(full, attention_masks=None)
    start = len(prompt_token_ids) - 1
    stop = start + len(gen_token_ids)
    return token_log_probs(logits[0, start:stop, :], full[0, start + 1:stop + 1])


def compute_policy_gradient_loss(model: torch.nn.Module, vllm_token_ids: list[list[int]],
                                 prompt_token_ids: list[list[int]], advantages: torch.Tensor,
                                 ref_token_log_probs: list[torch.Tensor], kl_coef: float = 0.1,
                                 ppo_clip_eps: float = 0.2, entropy_coef: float = 0.01):
    """(total loss, metrics dict, per-sample policy log-probs).

    Per sample: mean over its tokens of log(pi / pi_ref) -> ratio; clipped PPO objective on that
    ratio; KL by the k3 estimator ratio - 1 - log ratio per token, averaged per sample, then over
    samples; entropy bonus from the mean log-probability of all tokens."""
    device = next(model.parameters()).device
    advantages = advantages.to(device)
    batch_lps = [compute_token_log_probs(model, p, g, device) for p, g in zip(prompt_token_ids, vllm_token_ids)]
    numbers = (kl_coef, ppo_clip_eps, entropy_coef)
    if all(isinstance(x, (int, float)) for x in numbers) and ppo_clip_eps >= 0 and _one_launch(batch_lps, ref_token_log_probs, advantages):
        offsets = torch.tensor([0, *(lps.numel() for lps in batch_lps)], dtype=torch.int64).cumsum(0).to(device)
        ref = torch.cat(list(ref_token_log_probs))
        total, values = _sample_loss(torch.cat(batch_lps), advantages, ref, offsets, ppo_clip_eps, kl_coef, entropy_coef)
        return total, dict(zip(POLICY_METRICS, values.tolist())), batch_lps
    mean_log_ratio, mean_kl = [], []
    for lps, ref in zip(batch_lps, ref_token_log_probs):
        log_ratio = lps - ref.detach()
        mean_log_ratio.append(log_ratio.mean())
        mean_kl.append((torch.exp(log_ratio) - 1 - log_ratio).mean())
    mean_log_ratio, mean_kl = torch.stack(mean_log_ratio), torch.stack(mean_kl)
    ratio = torch.exp(mean_log_ratio)
    clipped_ratio = torch.clamp(ratio, 1 - ppo_clip_eps, 1 + ppo_clip_eps)
    pg_loss = -torch.min(ratio * advantages, clipped_ratio * advantages).mean()
    entropy = -torch.cat(batch_lps).mean()
    kl_div = mean_kl.mean()
    total = pg_loss + (-entropy_coef * entropy) + kl_coef * kl_div
    metrics = {
        "pg_loss": pg_loss.item(),
        "entropy": entropy.item(),
        "kl_div": kl_div.item(),
        "ratio_mean": ratio.mean().item(),
        "ratio_clipped_frac": (torch.abs(ratio - clipped_ratio) > 1e-6).float().mean().item(),
    }
    return total, metrics, batch_lps


def _one_launch(log_probs, ref, advantages: torch.Tensor) -> bool:
    """The samples' losses can be formed over all tokens at once: float32 on one GPU, no sample empty, outside function transforms."""
    if not log_probs or not (torch.compiler.is_compiling() or ops.plain_rows(log_probs[0])):
        return False
    plain = lambda t: type(t) is torch.Tensor and t.is_cuda and t.dtype == torch.float32 and t.device == advantages.device
    return (len(log_probs) == len(ref) and plain(advantages) and advantages.shape == (len(log_probs),)
            and not advantages.requires_grad
            and all(plain(a) and plain(b) and a.dim() == 1 and a.shape == b.shape and a.numel() > 0 for a, b in zip(log_probs, ref)))


POLICY_METRICS = ("pg_loss", "kl_div", "entropy", "ratio_mean", "ratio_clipped_frac")
_KL = ("k1", "k2", "k3", "k3_swapped")
_PREFERENCES = ("sigmoid", "hinge", "ipo")


def _check_tokens(log_probs, others: dict, offsets, mask) -> int:
    """How many sequences the tokens are of."""
    if not log_probs.is_floating_point():
        raise TypeError(f"log_probs must be floating-point, got {log_probs.dtype}")
    if log_probs.dim() != (2 if offsets is None else 1):
        raise ValueError(f"log_probs must be [sequences, length], or [tokens] with offsets; got {tuple(log_probs.shape)}"
                         f"{'' if offsets is None else ' with offsets'}")
    for name, t in others.items():
        if t is not None and not t.is_floating_point():
            raise TypeError(f"{name} must be floating-point, got {t.dtype}")
        if t is not None and t.shape != log_probs.shape:
            raise ValueError(f"{name} must have the shape of log_probs, {tuple(log_probs.shape)}, got {tuple(t.shape)}")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != log_probs.shape):
        raise ValueError(f"mask must be bool with the shape of log_probs, {tuple(log_probs.shape)}, got {tuple(mask.shape)} {mask.dtype}")
    if offsets is not None and (offsets.dtype not in (torch.int64, torch.int32) or offsets.dim() != 1 or offsets.numel() == 0):
        raise ValueError(f"offsets must be int64 or int32 [sequences + 1], got {tuple(offsets.shape)} {offsets.dtype}")
    for name, t in (*others.items(), ("offsets", offsets), ("mask", mask)):
        if t is not None and t.device != log_probs.device:
            raise ValueError(f"log_probs on {log_probs.device}, {name} on {t.device}")
    return log_probs.shape[0] if offsets is None else offsets.numel() - 1


def _once(grad):
    """A gradient that cannot be differentiated again: what it was formed from is in it."""
    return _Refusing.apply(grad, torch.empty(0, requires_grad=True)) if torch.is_grad_enabled() else grad


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, log_probs, *rest):
        loss, metrics, each = ops.policy_loss_fwd(log_probs, *rest)
        ctx.save_for_backward(log_probs, *rest[:5], each)
        ctx.numbers = rest[5:]
        ctx.mark_non_differentiable(metrics)
        return loss, metrics

    @staticmethod
    def backward(ctx, dloss, _):
        return (_once(ops.policy_loss_bwd(*ctx.saved_tensors, dloss, *ctx.numbers)), *(None,) * 14)


class _SampleLoss(_PolicyLoss):
    """The policy loss with a gradient that has one itself: where it is asked for, it is formed in torch operations."""

    @staticmethod
    def backward(ctx, dloss, _):
        if not torch.is_grad_enabled():
            return _PolicyLoss.backward(ctx, dloss, _)
        tensors = ctx.saved_tensors[:6]
        loss, _ = _policy_in_torch_ops(*tensors, *ctx.numbers)
        return (*torch.autograd.grad(loss, tensors[0], dloss, create_graph=True), *(None,) * 14)


def _sample_loss(log_probs, advantages, ref, offsets, clip_eps: float, kl_coef: float, entropy_coef: float):
    """(loss, metrics) with a ratio and a mean for each sample."""
    if torch.compiler.is_compiling():
        return policy_loss(log_probs, advantages, ref, ref, offsets=offsets, clip_eps=clip_eps, kl_coef=kl_coef, kl="k3_swapped",
                           entropy_coef=entropy_coef, ratio="sequence", average="sequence")
    return _SampleLoss.apply(log_probs, _dense(advantages), ref, ref, offsets, None, advantages.shape[0], False, True, True,
                             _KL.index("k3_swapped"), 1.0 - float(clip_eps), 1.0 + float(clip_eps), float(kl_coef), float(entropy_coef))


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, log_probs, *rest):
        loss, rewards, each = ops.preference_loss_fwd(log_probs, *rest)
        ctx.save_for_backward(log_probs, *rest[:3], each)
        ctx.numbers = rest[3:]
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    def backward(ctx, dloss, _):
        return (_once(ops.preference_loss_bwd(*ctx.saved_tensors, dloss, *ctx.numbers)), *(None,) * 8)


def _by_kernels(name: str, node, log_probs, tensors: tuple, numbers: tuple):
    """The loss through the kernels -- one native call, a traced operator, or step by step --, None for tensors that they do
    not take."""
    given = tuple(t for t in tensors if t is not None)
    if not log_probs.is_cuda or log_probs.dtype not in ops.ROW_TYPES or ops.wrapped(log_probs, *given):
        return None
    if any(t.dtype == torch.float64 for t in given):  # (the kernels would read it in float32)
        return None
    if torch.compiler.is_compiling():
        from .. import compiled  # noqa: F401  (the same launches as nodes of the graph)

        call = getattr(torch.ops.torchtitan_amd, name + "_fwd")
        loss, more, _ = call(log_probs, *(_wide(t) for t in tensors), *numbers)
        return loss, more.detach()  # (as the nodes mark it)
    if not ops.plain_rows(log_probs) or not all(type(t) in (torch.Tensor, torch.nn.Parameter) for t in given):
        return None
    if ops.native_rows(log_probs):
        call = getattr(_lib.blocks(), name)
        out = call(log_probs, *tensors, *numbers)
        if out is None:
            with torch.cuda.device(log_probs.device):
                out = call(log_probs.contiguous(), *(_dense(t) for t in tensors), *numbers)
        if out is not None:
            return out
    tensors = tuple(_dense(t) for t in tensors)
    if torch.is_grad_enabled() and log_probs.requires_grad:
        return node.apply(log_probs, *tensors, *numbers)
    return getattr(ops, name + "_fwd")(log_probs, *tensors, *numbers, want_each=False)[:2]


def _wide(t):
    """In a type that the kernels read, which holds all of its values."""
    return t.float() if t is not None and t.is_floating_point() and t.dtype not in ops.ROW_TYPES else t


def _dense(t):
    """Without a gradient, as the kernels read it and a node keeps it."""
    if t is None:
        return None
    t = _wide(t.detach()).resolve_neg().contiguous()
    return t.clone() if t.is_inference() else t


def _places(log_probs, offsets, mask, sequences: int):
    """(sequence of every token, whether it counts), flat."""
    place = torch.arange(log_probs.numel(), device=log_probs.device)
    if offsets is None:
        sequence = place // max(1, log_probs.shape[1])
        counts = torch.ones_like(place, dtype=torch.bool)
    else:
        sequence = torch.bucketize(place, offsets.long(), right=True) - 1
        counts = (sequence >= 0) & (sequence < sequences)
        sequence = sequence.clamp(0, max(0, sequences - 1))
    return sequence, counts if mask is None else counts & mask.reshape(-1)


def _sums(values, sequence, sequences: int):
    return values.new_zeros(sequences).index_add(0, sequence, values)


def _nothing(log_probs):
    """The loss of no sequences, with its gradient."""
    return log_probs[:0].float().sum()


def _kl_term(x, kind: int):
    if _KL[kind] == "k1":
        return x
    if _KL[kind] == "k2":
        return 0.5 * x * x
    if _KL[kind] == "k3":
        x = -x
    return torch.expm1(x) - x.clamp(max=1e300)  # (infinite where x is)


def _policy_in_torch_ops(log_probs, advantages, old, ref, offsets, mask, sequences, per_token, whole, by_sequence, kl, low, high,
                         kl_coef, entropy_coef):
    if sequences == 0:
        return _nothing(log_probs), torch.zeros(5, device=log_probs.device)
    sequence, counts = _places(log_probs, offsets, mask, sequences)
    flat = lambda t: torch.where(counts, t.reshape(-1).double(), 0.0)
    lp = flat(log_probs)
    n = _sums(counts.double(), sequence, sequences)
    tokens, filled, per_sequence = n.sum().clamp(min=1), (n > 0).sum().clamp(min=1).double(), n.clamp(min=1)
    each = (1 / (filled * per_sequence))[sequence] if by_sequence else (1 / tokens).expand_as(lp)
    x = lp - (lp.detach() if old is None else flat(old))
    A = advantages.detach().double()
    A = A.reshape(-1) if per_token else A[sequence]
    if whole:
        x = (_sums(x, sequence, sequences) / per_sequence)[sequence]
    A = torch.where(counts, A, 0.0)
    ratio = torch.exp(torch.where(A >= 0, x.detach(), x))
    # (where the upper border is behind, nothing that overflows is differentiated)
    bounded = torch.where(A >= 0, torch.exp(x.clamp(max=math.log(max(high, 1e-300)) + 1.0)).clamp(max=high), ratio.clamp(min=low))
    objective = -A * bounded
    mean = lambda values, weight: torch.where(counts, values * weight, 0.0).sum()
    pg, kl_div = mean(objective, each), lp.new_zeros(())
    if ref is not None:
        kl_div = mean(_kl_term(lp - flat(ref), kl), each)
    entropy = -lp.sum() / tokens
    total = pg + (kl_coef * kl_div if kl_coef else 0.0) - (entropy_coef * entropy if entropy_coef else 0.0)
    with torch.no_grad():
        per = (1 / (filled * per_sequence))[sequence] if whole else (1 / tokens).expand_as(lp)
        clipped = ((ratio - ratio.clamp(low, high)).abs() > 1e-6).double()
        metrics = torch.stack([pg.detach(), kl_div.detach(), entropy.detach(), mean(ratio, per), mean(clipped, per)]).float()
    return total.float(), metrics


def policy_loss(log_probs: torch.Tensor, advantages: torch.Tensor, old_log_probs: torch.Tensor | None = None,
                ref_log_probs: torch.Tensor | None = None, *, offsets: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                clip_eps: float = 0.2, clip_eps_high: float | None = None, kl_coef: float = 0.0, kl: str = "k3",
                entropy_coef: float = 0.0, ratio: str = "token", average: str = "token", advantage: str | None = None):
    """(loss, metrics): the clipped policy loss of many sequences, and float32 [5] metrics named by `POLICY_METRICS`.

        r = exp(log_probs - old_log_probs)       (or ratio="sequence": of the mean of that over a sequence)
        pg = mean of -min(r A, clip(r, 1 - clip_eps, 1 + clip_eps_high) A)
        loss = pg + kl_coef * (mean of the KL estimator) - entropy_coef * entropy

    log_probs: of the sampled tokens, [sequences, length], or [tokens] with `offsets` (int64 or int32 [sequences + 1]: sequence s has
    the tokens from offsets[s] to offsets[s + 1]; rising, not behind the last token).  `mask` (bool) says which of them count.  What a token
    that does not count holds has no influence, and its gradient is 0; sequences without a token that counts are left out of
    every mean.  advantages: [sequences], or of every token (ratio="token"); their shape says which, but for packed tokens as many as
    there are sequences, where `advantage`, "sequence" or "token", must (on the GPU they are read in float32, whatever their type).
    Without `old_log_probs` the policy has not moved: r is 1, with its gradient.  kl, at x = log_probs - ref_log_probs: "k1" x, "k2"
    x^2 / 2, "k3" exp(-x) - 1 + x, "k3_swapped" exp(x) - 1 - x.
    The entropy is minus the mean of log_probs.  average: means of pg and KL over all tokens, or over sequences of the means
    over their tokens.  A coefficient of 0 leaves its term out of the loss, whatever it is.  Only log_probs gets a gradient, which on the GPU
    cannot be differentiated again; terms and sums are in float64."""
    if ratio not in ("token", "sequence") or average not in ("token", "sequence"):
        raise ValueError(f"ratio and average must be 'token' or 'sequence', got {ratio!r} and {average!r}")
    if kl not in _KL:
        raise ValueError(f"kl must be one of {_KL}, got {kl!r}")
    if kl_coef and ref_log_probs is None:
        raise ValueError("kl_coef wants ref_log_probs")
    low, high = 1.0 - float(clip_eps), 1.0 + float(clip_eps if clip_eps_high is None else clip_eps_high)
    if not low <= high:
        raise ValueError(f"clip_eps {clip_eps} and clip_eps_high {clip_eps_high} leave nothing between them")
    sequences = _check_tokens(log_probs, dict(old_log_probs=old_log_probs, ref_log_probs=ref_log_probs), offsets, mask)
    if advantage not in (None, "token", "sequence") or (advantage == "token" and ratio == "sequence"):
        raise ValueError(f"advantage must be 'sequence', or 'token' with ratio='token', got {advantage!r} with {ratio!r}")
    per_token = advantages.shape != (sequences,) if advantage is None else advantage == "token"
    if advantage is None and ratio == "token" and advantages.shape == log_probs.shape == (sequences,) and sequences > 1:
        raise ValueError(f"{sequences} packed tokens of {sequences} sequences: advantage='sequence' or advantage='token' has to say what "
                         "the advantages belong to")
    if (advantages.shape != (log_probs.shape if per_token else (sequences,)) or (per_token and ratio == "sequence")
            or not advantages.is_floating_point()):
        raise ValueError(f"advantages must be floating-point [{sequences}]{'' if ratio == 'sequence' else f' or {tuple(log_probs.shape)}'}, "
                         f"got {tuple(advantages.shape)} {advantages.dtype}")
    if advantages.device != log_probs.device:
        raise ValueError(f"log_probs on {log_probs.device}, advantages on {advantages.device}")
    numbers = (sequences, per_token, ratio == "sequence", average == "sequence", _KL.index(kl), low, high, float(kl_coef),
               float(entropy_coef))
    out = _by_kernels("policy_loss", _PolicyLoss, log_probs,
                      (advantages if advantages.dtype == torch.float32 else advantages.float(), old_log_probs, ref_log_probs, offsets,
                       mask), numbers)
    if out is not None:
        return out
    return _policy_in_torch_ops(log_probs, advantages, old_log_probs if old_log_probs is None else old_log_probs.detach(),
                                ref_log_probs if ref_log_probs is None else ref_log_probs.detach(), offsets, mask, *numbers)


def _preference_in_torch_ops(log_probs, ref, offsets, mask, sequences, kind, mean, beta, smoothing):
    if sequences == 0:
        return _nothing(log_probs), torch.zeros(0, device=log_probs.device)
    sequence, counts = _places(log_probs, offsets, mask, sequences)
    flat = lambda t: torch.where(counts, t.reshape(-1).double(), 0.0)
    x = flat(log_probs) if ref is None else flat(log_probs) - flat(ref)
    n = _sums(counts.double(), sequence, sequences)
    h = _sums(x, sequence, sequences)
    if mean:
        h = h / n.clamp(min=1)
    z, pairs = h[:sequences // 2] - h[sequences // 2:], n[:sequences // 2] + n[sequences // 2:] > 0
    if _PREFERENCES[kind] == "sigmoid":
        losses = -(1 - smoothing) * F.logsigmoid(beta * z)
        if smoothing:  # (a part of 0 would be no number where z is infinite)
            losses = losses - smoothing * F.logsigmoid(-beta * z)
    elif _PREFERENCES[kind] == "hinge":
        losses = F.relu(1 - beta * z)
    else:
        losses = (z - 0.5 / beta) ** 2
    loss = torch.where(pairs, losses, 0.0).sum() / pairs.sum().clamp(min=1)
    return loss.float(), (beta * h.detach()).float()


def preference_loss(log_probs: torch.Tensor, ref_log_probs: torch.Tensor | None = None, *, offsets: torch.Tensor | None = None,
                    mask: torch.Tensor | None = None, beta: float = 0.1, kind: str = "sigmoid", label_smoothing: float = 0.0,
                    average_log_probs: bool = False):
    """(loss, rewards): the preference loss of pairs of sequences, and float32 [sequences] rewards beta * h.

        h = sum over a sequence's tokens of log_probs - ref_log_probs     (their mean with `average_log_probs`)
        z = h of the preferred sequence - h of the other
        "sigmoid": -(1 - label_smoothing) log sigmoid(beta z) - label_smoothing log sigmoid(-beta z)
        "hinge":   max(0, 1 - beta z)              "ipo": (z - 1 / (2 beta))^2

    averaged over the pairs.  The first half of the sequences are the preferred ones, the second half the others, in the same
    order.  Tokens, `offsets` and `mask` as for ``policy_loss``; a pair without a token that counts is left out, and a sequence without
    one beside an answer that has some has h = 0.  Without
    `ref_log_probs` h is of log_probs alone.  Only log_probs gets a gradient, which on the GPU cannot be differentiated
    again; terms and sums are in float64."""
    if kind not in _PREFERENCES:
        raise ValueError(f"kind must be one of {_PREFERENCES}, got {kind!r}")
    if not beta > 0:
        raise ValueError(f"beta must be positive, got {beta}")
    if not 0 <= label_smoothing <= 0.5 or (label_smoothing and kind != "sigmoid"):
        raise ValueError(f"label_smoothing is of the sigmoid loss, from 0 to 0.5; got {label_smoothing} with {kind!r}")
    sequences = _check_tokens(log_probs, dict(ref_log_probs=ref_log_probs), offsets, mask)
    if sequences % 2:
        raise ValueError(f"pairs want an even number of sequences, got {sequences}")
    numbers = (sequences, _PREFERENCES.index(kind), bool(average_log_probs), float(beta), float(label_smoothing))
    out = _by_kernels("preference_loss", _PreferenceLoss, log_probs, (ref_log_probs, offsets, mask), numbers)
    if out is not None:
        return out
    return _preference_in_torch_ops(log_probs, ref_log_probs if ref_log_probs is None else ref_log_probs.detach(), offsets, mask,
                                    *numbers)
