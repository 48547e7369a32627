"""GPU: gradients of the gradients of the sample loss."""
import pytest
import torch

from torchtitan_amd.rl import compute_policy_gradient_loss

pytestmark = pytest.mark.gpu


class Table(torch.nn.Module):
    """Logits of the next token, in the parameter's type."""

    def __init__(self, dtype, device):
        super().__init__()
        self.table = torch.nn.Parameter(torch.randn(50, 50, generator=torch.Generator().manual_seed(0)).to(device, dtype))

    def forward(self, tokens, attention_masks=None):
        return self.table[tokens]


PROMPTS, ANSWERS = [[1, 2], [3], [4, 5, 6]], [[7, 8, 9], [10], [11, 12, 13, 14]]
ADVANTAGES = [1.0, -0.5, 0.25]


def reference64(table, ref, direction, kl_coef, eps, entropy_coef):
    """(loss, its gradient, the gradient of that gradient along `direction`) in 64 bits."""
    table = table.detach().double().cpu().requires_grad_(True)
    pg, kl, lps = [], [], []
    for prompt, answer, r, A in zip(PROMPTS, ANSWERS, ref, ADVANTAGES):
        before = torch.tensor([prompt[-1], *answer[:-1]])
        lp = torch.log_softmax(table[before], -1)[torch.arange(len(answer)), torch.tensor(answer)]
        x = lp - r.double().cpu()
        ratio = x.mean().exp()
        pg.append(-torch.minimum(ratio * A, ratio.clamp(1 - eps, 1 + eps) * A))
        kl.append((x.exp() - 1 - x).mean())
        lps.append(lp)
    loss = torch.stack(pg).mean() + kl_coef * torch.stack(kl).mean() + entropy_coef * torch.cat(lps).mean()
    (g,) = torch.autograd.grad(loss, table, create_graph=True)
    (gg,) = torch.autograd.grad((g * direction.double().cpu()).sum(), table)
    return loss.detach(), g.detach(), gg


@pytest.mark.parametrize("kl_coef,eps,entropy_coef", [(0.1, 0.2, 0.01), (0.0, 5.0, 0.0), (0.3, 5.0, 0.1)])
def test_a_float32_model_can_be_differentiated_twice(device, kl_coef, eps, entropy_coef):
    model = Table(torch.float32, device)
    ref = [(torch.randn(len(a), generator=torch.Generator().manual_seed(i)) * 0.3 - 4).to(device) for i, a in enumerate(ANSWERS)]
    direction = torch.randn(50, 50, generator=torch.Generator().manual_seed(9)).to(device)
    numbers = dict(kl_coef=kl_coef, ppo_clip_eps=eps, entropy_coef=entropy_coef)
    total, metrics, lps = compute_policy_gradient_loss(model, ANSWERS, PROMPTS, torch.tensor(ADVANTAGES), ref, **numbers)
    (once,) = torch.autograd.grad(total, model.table, retain_graph=True)
    (g,) = torch.autograd.grad(total, model.table, create_graph=True)
    (gg,) = torch.autograd.grad((g * direction).sum(), model.table, retain_graph=True)
    loss64, g64, gg64 = reference64(model.table, ref, direction, kl_coef, eps, entropy_coef)
    # log-probabilities of up to 8 in float32: a log-softmax is off by some 10 roundings of that, 8e-5 * 2^-4 = 5e-6, which is the
    # relative error of every ratio and probability in a term; terms are at most the largest second derivative and gradient
    for got, want in ((total.detach(), loss64), (once, g64), (g.detach(), g64), (gg, gg64)):
        assert float((got.double().cpu() - want).abs().max()) <= 3e-5 * float(want.abs().max() + g64.abs().max())
    # (a penalty on the gradient, as a training step forms it)
    penalty = total + (g * g).sum()
    penalty.backward()
    assert torch.isfinite(model.table.grad).all()


def test_a_bf16_model_refuses_it(device):
    """Its log-probabilities' kernel has a gradient without one of its own."""
    model = Table(torch.bfloat16, device)
    ref = [torch.full((len(a),), -4.0, device=device) for a in ANSWERS]
    total = compute_policy_gradient_loss(model, ANSWERS, PROMPTS, torch.tensor(ADVANTAGES), ref)[0]
    (g,) = torch.autograd.grad(total, model.table, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        g.float().square().sum().backward()
