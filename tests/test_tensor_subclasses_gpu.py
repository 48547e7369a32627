"""Embedding, norms and clipping of tensors that are more than their values."""
import pytest
import torch

from torchtitan_amd import _lib, ops
from torchtitan_amd.gradients import clip_grad_norm_, get_total_norm
from torchtitan_amd.modules import residual_rms_norm, scaled_embedding

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


class Named(torch.Tensor):
    """No operation of its own: torch's operations keep the type."""


class Watching(torch.Tensor):
    seen = 0

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        cls.seen += 1
        return super().__torch_function__(func, types, args, kwargs or {})


@pytest.mark.parametrize("cls", [Named, Watching])
def test_subclasses_keep_their_type(device, cls):
    """In any place of the call, with gradients and without, the result is what the formula in torch operations makes of it."""
    plain = lambda *s: torch.randn(s, device=device).to(BF)
    ids = torch.randint(0, 9, (5,), device=device)
    weight = plain(9, 16)
    want = scaled_embedding(ids, weight, 2.0)
    for grad in (False, True):
        w = weight.clone().as_subclass(cls).requires_grad_(grad)
        for out in (scaled_embedding(ids, w, 2.0), scaled_embedding(ids.as_subclass(cls), weight.clone().requires_grad_(grad), 2.0)):
            assert type(out) is cls and torch.equal(out.as_subclass(torch.Tensor), want)
    operands = dict(h=plain(4, 64), residual=plain(4, 64), post_weight=plain(64), gate=plain(64), pre_weight=plain(64))
    want = residual_rms_norm(**operands)
    for name in operands:
        for grad in (False, True):
            with_one = {k: v.clone().requires_grad_(grad) for k, v in operands.items()}
            with_one[name] = operands[name].clone().as_subclass(cls).requires_grad_(grad)
            out = residual_rms_norm(**with_one)
            assert type(out[1]) is cls and (type(out[0]) is cls or name == "pre_weight"), name
            # the same formula in float32, its sums in another order: a step of bf16 of the largest value
            assert all((a.as_subclass(torch.Tensor).float() - b.float()).abs().max() <= 2.0 ** -7 * b.abs().max() for a, b in zip(out, want))


def test_subclasses_of_gradients(device):
    p, q = (torch.nn.Parameter(torch.zeros(40, device=device)) for _ in range(2))
    p.grad, q.grad = torch.randn(40, device=device), torch.randn(40, device=device).as_subclass(Watching)
    exact = float(p.grad.double().square().sum() + q.grad.as_subclass(torch.Tensor).double().square().sum()) ** 0.5
    before, Watching.seen = q.grad.as_subclass(torch.Tensor).clone(), 0
    norm = clip_grad_norm_([p, q], exact / 2)
    assert Watching.seen > 0
    assert abs(float(norm) - exact) <= 1e-6 * exact  # 80 squares in float32
    assert (q.grad.as_subclass(torch.Tensor) - before / 2).abs().max() <= 1e-5 * before.abs().max()


def test_plain_tensors_and_parameters_take_the_native_call(device):
    native = _lib.blocks()
    ids = torch.randint(0, 9, (5,), device=device)
    weight = torch.nn.Parameter(torch.randn((9, 16), device=device))
    assert native.scaled_embedding(ids, weight, 2.0, None, 0, True) is not None
    assert native.scaled_embedding(ids, weight.detach(), 2.0, None, 0, True) is not None
    assert native.scaled_embedding(ids, weight.detach().as_subclass(Named), 2.0, None, 0, True) is None
    h = torch.randn((4, 16), device=device)
    assert native.residual_rms_norm(h, h * 2, weight[0].detach(), torch.nn.Parameter(h[0].clone()), None, 1.0, 1e-5) is not None
    assert native.residual_rms_norm(h, h * 2, weight[0].detach().as_subclass(Named), None, None, 1.0, 1e-5) is None
    weight.grad = torch.ones_like(weight)
    assert native.clip_gradients([weight], 1.0, 0) is not None
    (weight.square().sum()).backward()  # a gradient that no program has held yet
    assert native.clip_gradients([weight], 1.0, 0) is not None
    assert ops.plain_rows(weight, h)
    assert get_total_norm([weight.grad]).dtype == torch.float32
