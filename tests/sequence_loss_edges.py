"""Infinite values, equal shapes and wide operands in the policy and preference losses, on any device."""
import math

import pytest
import torch

from torchtitan_amd.rl import policy_loss, preference_loss


def a_rejected_answer_without_a_chance(device):
    """log p of the rejected sequence is minus infinity: nothing is lost on the pair, and it has no gradient."""
    lp = torch.tensor([[-1.0, -2.0], [-3.0, -1.0], [-math.inf, -1.0], [-1.5, -2.5]], device=device, requires_grad=True)
    loss, rewards = preference_loss(lp, beta=0.5)
    z = -4.0 + 4.0
    assert math.isclose(loss.item(), (0.0 + math.log1p(math.exp(-0.5 * z))) / 2, rel_tol=1e-6)
    assert rewards.tolist()[2] == -math.inf
    (grad,) = torch.autograd.grad(loss, lp)
    assert torch.equal(grad, torch.tensor([[0.0, 0.0], [-0.125, -0.125], [0.0, 0.0], [0.125, 0.125]], device=device))
    for kind in ("hinge", "sigmoid"):  # (the other way round it is infinite)
        swapped = torch.cat((lp[2:], lp[:2])).detach().requires_grad_(True)
        assert preference_loss(swapped, beta=0.5, kind=kind)[0].item() == math.inf
    assert preference_loss(lp, beta=0.5, label_smoothing=0.1)[0].item() == math.inf


def a_token_that_the_reference_rules_out(device):
    """The estimators at x = +inf and -inf: infinite, with the sign of their gradient."""
    lp = torch.tensor([[-1.0, -2.0]], device=device, requires_grad=True)
    for kl, value, slope in (("k1", math.inf, 1.0), ("k2", math.inf, math.inf), ("k3", math.inf, 1.0), ("k3_swapped", math.inf, math.inf)):
        loss, metrics = policy_loss(lp, torch.zeros(1, device=device), None, torch.tensor([[-1.0, -math.inf]], device=device), kl=kl,
                                    kl_coef=1.0)
        assert loss.item() == value and metrics[1].item() == value, kl
        (grad,) = torch.autograd.grad(loss, lp)
        assert grad[0, 1].item() == slope / 2, kl
    for kl, value in (("k1", -math.inf), ("k2", math.inf), ("k3", math.inf), ("k3_swapped", math.inf)):
        _, metrics = policy_loss(torch.tensor([[-1.0, -math.inf]], device=device), torch.zeros(1, device=device),
                                 torch.zeros(1, 2, device=device), torch.tensor([[-1.0, -1.0]], device=device), kl=kl)
        assert metrics[1].item() == value, kl


def as_many_tokens_as_sequences(device):
    """Packed, the shape of the advantages does not say what they belong to."""
    lp = torch.zeros(4, device=device, requires_grad=True)
    A = torch.tensor([1.0, 2.0, 3.0, 4.0], device=device)
    for bounds, by_token, by_sequence in (([0, 3, 3, 3, 4], [1.0, 2.0, 3.0, 4.0], [1.0, 1.0, 1.0, 4.0]),
                                          ([0, 1, 1, 2, 2], [1.0, 2.0, 0.0, 0.0], [1.0, 3.0, 0.0, 0.0]),
                                          ([0, 1, 2, 3, 4], [1.0, 2.0, 3.0, 4.0], [1.0, 2.0, 3.0, 4.0])):
        offsets = torch.tensor(bounds, device=device)
        with pytest.raises(ValueError, match="advantage="):
            policy_loss(lp, A, offsets=offsets)
        for advantage, want in (("token", by_token), ("sequence", by_sequence)):
            loss, _ = policy_loss(lp, A, offsets=offsets, advantage=advantage)
            n = bounds[-1]
            assert math.isclose(loss.item(), -sum(want) / n, rel_tol=1e-6)
            (grad,) = torch.autograd.grad(loss, lp)
            assert torch.allclose(grad, -torch.tensor(want, device=device) / n, rtol=1e-6)
        # (a ratio of a sequence has the sequence's advantage)
        assert math.isclose(policy_loss(lp, A, offsets=offsets, ratio="sequence")[0].item(), -sum(by_sequence) / n, rel_tol=1e-6)
    one = policy_loss(lp[:1], A[:1], offsets=torch.tensor([0, 1], device=device))[0]
    assert one.item() == -1.0  # (one token of one sequence: the same)
    rows = torch.zeros(4, 1, device=device)
    assert policy_loss(rows, A)[0].item() == policy_loss(rows, A[:, None])[0].item() == -2.5
    for bad, wrong in ((dict(advantage="row"), A), (dict(advantage="token", ratio="sequence"), A[:, None]), (dict(advantage="token"), A),
                       (dict(advantage="sequence"), A[:, None])):
        with pytest.raises(ValueError):
            policy_loss(rows, wrong, **bad)


def a_border_between_two_float32_numbers(device):
    """Old log-probabilities in float64: ratios on either side of a border, nearer to it than float32 tells."""
    border = -math.log(1.2)
    lp = torch.zeros(1, 2, device=device, requires_grad=True)
    old = torch.tensor([[border - 1e-10, border + 1e-10]], dtype=torch.float64, device=device)
    loss, metrics = policy_loss(lp, torch.ones(1, device=device), old, clip_eps=0.2)
    (grad,) = torch.autograd.grad(loss, lp)
    assert grad[0, 0].item() == 0.0 and abs(grad[0, 1].item() + 0.6) <= 1e-6
    # and a reference: 1e-9 between the two of a pair
    pair = torch.full((2, 1), -2.0, device=device, requires_grad=True)
    ref = torch.tensor([[-2.0 - 1e-9], [-2.0 + 1e-9]], dtype=torch.float64, device=device)
    _, rewards = preference_loss(pair, ref, beta=1.0)
    assert all(abs(a - b) <= 1e-15 for a, b in zip(rewards.tolist(), (1e-9, -1e-9)))
    x = torch.full((1, 1), 1e-9, dtype=torch.float64, device=device)
    _, metrics = policy_loss(pair[:1], torch.ones(1, device=device), None, pair[:1].double().detach() - x, kl="k1")
    assert abs(metrics[1].item() - 1e-9) <= 1e-15


def operands_from_inference_mode(device):
    """What a rollout computed in inference mode is an operand like any other."""
    lp = torch.full((3, 4), -1.0, device=device, requires_grad=True)
    with torch.inference_mode():
        old, ref = (torch.full((3, 4), v, device=device) for v in (-1.25, -1.5))
        A, mask = torch.ones(3, device=device), torch.ones(3, 4, dtype=torch.bool, device=device)
    plain = [t.clone() for t in (A, old, ref, mask)]
    for make in (lambda A, old, ref, mask: policy_loss(lp, A, old, ref, mask=mask, kl_coef=0.1)[0],
                 lambda A, old, ref, mask: preference_loss(torch.cat((lp, lp * 2)), torch.cat((ref, old)), mask=torch.cat((mask, mask)))[0],
                 lambda A, old, ref, mask: preference_loss(lp[:2], ref[:2], mask=mask[:2])[0]):
        got, want = make(A, old, ref, mask), make(*plain)
        assert torch.equal(got, want)
        assert torch.equal(torch.autograd.grad(got, lp)[0], torch.autograd.grad(want, lp)[0])
