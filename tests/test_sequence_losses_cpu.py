"""CPU: the policy and preference losses in torch operations against 64 bits, differences, and their refusals."""
import ctypes
import math

import pytest
import torch

from tests.sequence_losses import check_policy, check_preference, policy64, preference64, tokens_of
from torchtitan_amd import _lib
from torchtitan_amd.rl import POLICY_METRICS, compute_policy_gradient_loss, policy_loss, preference_loss

LAYOUTS = [dict(shape=(6, 9)), dict(shape=(6, 9), mask=0.6), dict(shape=(1, 1)), dict(shape=(4, 0)), dict(shape=(2, 70), mask=0.0),
           dict(shape=(60,), offsets=[0, 7, 7, 30, 60]), dict(shape=(60,), offsets=[3, 10, 11, 12, 55], mask=0.7),
           dict(shape=(5,), offsets=[0]), dict(shape=(0,), offsets=[0, 0, 0])]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("ratio", ["token", "sequence"])
@pytest.mark.parametrize("average", ["token", "sequence"])
def test_policy_loss_in_torch_operations(layout, ratio, average):
    for kl in ("k1", "k2", "k3", "k3_swapped"):
        check_policy(policy_loss, tokens_of(device="cpu", **layout), ratio=ratio, average=average, kl=kl, kl_coef=0.3, entropy_coef=0.1,
                     clip_eps=0.1, clip_eps_high=0.3)
    check_policy(policy_loss, tokens_of(device="cpu", old=False, ref=False, **layout), ratio=ratio, average=average)
    if ratio == "token":
        check_policy(policy_loss, tokens_of(device="cpu", per_token=True, dtype=torch.bfloat16, **layout), average=average)


@pytest.mark.parametrize("layout", [x for x in LAYOUTS if x["shape"] != (1, 1)])
@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("ipo", 0.0)])
def test_preference_loss_in_torch_operations(layout, kind, smoothing):
    for mean in (False, True):
        for dtype in (torch.float32, torch.bfloat16):
            check_preference(preference_loss, tokens_of(device="cpu", dtype=dtype, **layout), kind=kind, label_smoothing=smoothing,
                             average_log_probs=mean, beta=0.7)
    check_preference(preference_loss, tokens_of(device="cpu", ref=False, **layout), kind=kind, label_smoothing=smoothing)


def test_the_gradients_are_the_differences_of_the_losses():
    case = tokens_of((4, 5), "cpu", mask=0.8, dtype=torch.float64)
    for options in (dict(), dict(ratio="sequence", average="sequence"), dict(average="sequence", kl="k3_swapped")):
        options = dict(options, kl_coef=0.2, entropy_coef=0.1)
        gradient = policy64(case, **options)[2]
        for i in (0, 3, 7, 19):
            moved = []
            for d in (1e-6, -1e-6):
                shifted = dict(case, log_probs=case["log_probs"].detach().clone())
                shifted["log_probs"].view(-1)[i] += d
                moved.append(policy64(shifted, **options)[0])
            # central differences: 1e-12 of the third derivative, and rounding of the loss (1e-16) over 2e-6
            assert abs((moved[0] - moved[1]) / 2e-6 - gradient[i]) <= 1e-9
    for kind in ("sigmoid", "ipo"):
        gradient = preference64(case, kind=kind)[2]
        for i in (0, 6, 19):
            moved = []
            for d in (1e-6, -1e-6):
                shifted = dict(case, log_probs=case["log_probs"].detach().clone())
                shifted["log_probs"].view(-1)[i] += d
                moved.append(preference64(shifted, kind=kind)[0])
            assert abs((moved[0] - moved[1]) / 2e-6 - gradient[i]) <= 1e-7  # (losses of some tens: rounding 1e-15 over 2e-6)


def test_on_the_border_and_without_an_advantage():
    lp = torch.tensor([[0.0, 0.0, 0.0]], requires_grad=True)
    old = torch.tensor([[-math.log(2.0), 0.0, -800.0]])
    loss, metrics = policy_loss(lp, torch.tensor([[1.0, -1.0, 0.0]]), old, clip_eps=0.5, clip_eps_high=1.0)
    # (2 is on the upper border and has its gradient; exp(800) without an advantage is nothing)
    assert abs(float(loss) - (-2.0 + 1.0) / 3) <= 1e-7
    (grad,) = torch.autograd.grad(loss, lp)
    assert torch.allclose(grad, torch.tensor([[-2.0 / 3 if math.exp(float(lp[0, 0] - old[0, 0])) <= 2.0 else 0.0, 1.0 / 3, 0.0]]))


def test_the_reference_loss_is_a_case_of_it():
    """compute_policy_gradient_loss over samples is policy_loss over their tokens packed."""
    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.table = torch.nn.Parameter(torch.randn(50, 50, generator=torch.Generator().manual_seed(0)))

        def forward(self, tokens, attention_masks=None):
            return self.table[tokens]

    model = Model()
    prompts, answers = [[1, 2], [3], [4, 5, 6]], [[7, 8, 9], [10], [11, 12, 13, 14]]
    ref = [torch.randn(len(a), generator=torch.Generator().manual_seed(i)) - 4 for i, a in enumerate(answers)]
    advantages = torch.tensor([1.0, -0.5, 0.25])
    total, metrics, lps = compute_policy_gradient_loss(model, answers, prompts, advantages, ref)
    offsets = torch.tensor([0, 3, 4, 8])
    loss, values = policy_loss(torch.cat(lps), advantages, torch.cat(ref), torch.cat(ref), offsets=offsets, kl_coef=0.1,
                               kl="k3_swapped", entropy_coef=0.01, ratio="sequence", average="sequence")
    assert torch.allclose(loss, total, rtol=1e-6)  # (some ten float32 roundings)
    for name, value in zip(POLICY_METRICS, values.tolist()):
        assert math.isclose(value, metrics[name], rel_tol=1e-6, abs_tol=1e-7), name
    a, b = (torch.autograd.grad(t, model.table, retain_graph=True)[0] for t in (loss, total))
    assert torch.allclose(a, b, rtol=1e-5, atol=1e-7)


def overflowing_terms(device):
    """A KL term and an entropy that are infinite, with coefficients of 0 and without."""
    lp = torch.tensor([[0.0, -1.0, -math.inf]], device=device, requires_grad=True)
    ref = torch.tensor([[-800.0, -1.0, -math.inf]], device=device)
    loss, metrics = policy_loss(lp, torch.ones(1, device=device), None, ref, mask=torch.tensor([[True, True, False]], device=device),
                                kl="k3_swapped")
    assert loss.item() == -1.0 and math.isinf(metrics[1].item())
    assert torch.equal(torch.autograd.grad(loss, lp)[0], torch.tensor([[-0.5, -0.5, 0.0]], device=device))
    assert math.isinf(policy_loss(lp[:, :2], torch.ones(1, device=device), None, ref[:, :2], kl="k3_swapped", kl_coef=0.1)[0].item())


def test_terms_without_a_coefficient_are_left_out():
    overflowing_terms("cpu")


def test_refusals():
    lp = torch.zeros(4, 5)
    A = torch.zeros(4)
    for error, call in (
            (ValueError, lambda: policy_loss(lp, A, ratio="sample")), (ValueError, lambda: policy_loss(lp, A, average="all")),
            (ValueError, lambda: policy_loss(lp, A, lp, kl="k4")), (ValueError, lambda: policy_loss(lp, A, kl_coef=0.1)),
            (ValueError, lambda: policy_loss(lp, A, clip_eps=-0.3, clip_eps_high=0.1)),
            (ValueError, lambda: policy_loss(lp[0], A)), (ValueError, lambda: policy_loss(lp, A, offsets=torch.zeros(2).long())),
            (ValueError, lambda: policy_loss(lp[0], torch.zeros(1), offsets=torch.zeros(2))),
            (ValueError, lambda: policy_loss(lp[0], torch.zeros(1), offsets=torch.zeros(0).long())),
            (ValueError, lambda: policy_loss(lp, A[:3])), (ValueError, lambda: policy_loss(lp, lp, ratio="sequence")),
            (ValueError, lambda: policy_loss(lp, A.long())), (ValueError, lambda: policy_loss(lp, A, lp[:, :4])),
            (TypeError, lambda: policy_loss(lp.long(), A)), (TypeError, lambda: policy_loss(lp, A, lp.long())),
            (ValueError, lambda: policy_loss(lp, A, mask=lp)), (ValueError, lambda: policy_loss(lp, A, mask=lp[:, 1:] > 0)),
            (ValueError, lambda: policy_loss(lp, A.to("meta"))), (ValueError, lambda: policy_loss(lp, A, lp.to("meta"))),
            (ValueError, lambda: preference_loss(lp[:3])), (ValueError, lambda: preference_loss(lp, kind="none")),
            (ValueError, lambda: preference_loss(lp, beta=0.0)), (ValueError, lambda: preference_loss(lp, label_smoothing=0.6)),
            (ValueError, lambda: preference_loss(lp, kind="hinge", label_smoothing=0.1)),
            (ValueError, lambda: preference_loss(lp, lp[1:]))):
        with pytest.raises(error):
            call()


def test_entry_points_refuse_before_any_launch():
    lib = _lib.load()
    P = ctypes.c_void_p

    class Policy(ctypes.Structure):
        _fields_ = [("log_probs", P), ("old", P), ("ref", P), ("lp_f32", ctypes.c_int), ("old_f32", ctypes.c_int),
                    ("ref_f32", ctypes.c_int), ("advantages", P), ("offsets", P), ("mask", P), ("sequences", ctypes.c_int64),
                    ("tokens", ctypes.c_int64), ("length", ctypes.c_int64), ("wide", ctypes.c_int), ("per_token", ctypes.c_int),
                    ("whole", ctypes.c_int), ("by_sequence", ctypes.c_int), ("kl", ctypes.c_int), ("low", ctypes.c_double),
                    ("high", ctypes.c_double), ("kl_coef", ctypes.c_double), ("entropy_coef", ctypes.c_double)]

    class Preference(ctypes.Structure):
        _fields_ = [("log_probs", P), ("ref", P), ("lp_f32", ctypes.c_int), ("ref_f32", ctypes.c_int), ("offsets", P), ("mask", P),
                    ("sequences", ctypes.c_int64), ("tokens", ctypes.c_int64), ("length", ctypes.c_int64), ("wide", ctypes.c_int),
                    ("kind", ctypes.c_int), ("mean", ctypes.c_int), ("beta", ctypes.c_double), ("smoothing", ctypes.c_double)]

    good = dict(log_probs=0x1000, lp_f32=1, sequences=4, tokens=20, length=5)
    out = (P(0x2000), P(0x3000), P(0x4000), P(0x5000), None)
    policy = lambda args=None, out=out, **at: lib.mx_policy_loss(ctypes.byref(Policy(**dict(good, advantages=0x6000, **at))), *out)
    preference = lambda out=out, **at: lib.mx_preference_loss(ctypes.byref(Preference(**dict(good, beta=0.1, **at))), *out)
    for call in (policy, preference):
        change = lambda **at: call(**at)
        for bad in (dict(out=(None, *out[1:])), dict(out=(*out[:3], None, None))):
            assert change(**bad) == 1
        assert change(out=(P(0x2002), *out[1:])) == 2 and change(out=(*out[:2], P(0x4004), *out[3:])) == 2
    bad = lambda cls, fn, extra, **at: fn(ctypes.byref(cls(**{**good, **extra, **at})), *out)
    for cls, fn, extra in ((Policy, lib.mx_policy_loss, dict(advantages=0x6000)), (Preference, lib.mx_preference_loss, dict(beta=0.1))):
        for at in (dict(log_probs=None), dict(sequences=-1), dict(tokens=21), dict(sequences=0), dict(length=-5)):
            assert bad(cls, fn, extra, **at) == 1
        assert bad(cls, fn, extra, log_probs=0x1002) == 2 and bad(cls, fn, extra, offsets=0x7004, wide=1) == 2
        assert bad(cls, fn, extra, tokens=1 << 32, length=1 << 30) == 4
        assert bad(cls, fn, extra, sequences=1 << 30, tokens=0, length=0) == 4
    assert bad(Policy, lib.mx_policy_loss, {}) == 1 and bad(Policy, lib.mx_policy_loss, dict(advantages=0x6000), kl=4) == 1
    assert bad(Policy, lib.mx_policy_loss, dict(advantages=0x6000), whole=1, per_token=1) == 1
    assert bad(Preference, lib.mx_preference_loss, dict(beta=0.1), sequences=5, length=4) == 1
    assert bad(Preference, lib.mx_preference_loss, dict(beta=0.1), kind=3) == 1
    assert lib.mx_policy_loss(None, *out) == 1 and lib.mx_preference_loss(None, *out) == 1
    args = Policy(**dict(good, advantages=0x6000))
    assert lib.mx_policy_loss_bwd(ctypes.byref(args), None, P(0x2000), P(0x3000), None) == 1
    assert lib.mx_policy_loss_bwd(ctypes.byref(args), P(0x2000), P(0x3000), P(0x4002), None) == 2
    args = Policy(**dict(good, advantages=0x6000, tokens=0, length=0))
    assert lib.mx_policy_loss_bwd(ctypes.byref(args), None, None, None, None) == 0
    assert lib.mx_sequence_loss_workspace(0, 0) > 0 and lib.mx_sequence_loss_workspace(1 << 20, 4096) < 1 << 20
