"""GPU: a gradient of the gradient of the fused token log-probabilities."""
import pytest
import torch

from torchtitan_amd.rl import token_log_probs

pytestmark = pytest.mark.gpu


def test_log_probs_of_bf16_logits_refuse_a_second_derivative(device):
    """Their kernel's gradient has no gradient of its own; without an error a penalty would miss it."""
    logits = torch.randn(12, 200, device=device).bfloat16().requires_grad_(True)
    lp = token_log_probs(logits, torch.arange(12, device=device))
    (g,) = torch.autograd.grad((lp * lp).sum(), logits, create_graph=True)
    (plain,) = torch.autograd.grad((lambda t: (t * t).sum())(token_log_probs(logits, torch.arange(12, device=device))), logits)
    assert torch.equal(g, plain)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        g.float().square().sum().backward()
