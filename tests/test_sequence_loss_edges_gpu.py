"""GPU: the losses' edges in the kernels, and traced."""
import pytest
import torch

from tests import sequence_loss_edges as edges
from tests.sequence_losses import tokens_of
from torchtitan_amd.rl import policy_loss, preference_loss

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", ["a_rejected_answer_without_a_chance", "a_token_that_the_reference_rules_out",
                                  "as_many_tokens_as_sequences", "a_border_between_two_float32_numbers", "operands_from_inference_mode"])
def test_edge(device, case):
    getattr(edges, case)(device)


def test_what_is_measured_has_no_gradient_in_a_graph_either(device):
    """Metrics and rewards of a traced call are as the eager ones: numbers to read."""
    case = tokens_of((8, 40), device, mask=0.7)

    def call(lp):
        loss, metrics = policy_loss(lp, case["advantages"], case["old"], case["ref"], mask=case["mask"], kl_coef=0.1)
        other, rewards = preference_loss(lp, case["ref"], mask=case["mask"])
        return loss, other, metrics, rewards

    torch._dynamo.reset()
    try:
        for traced in (call, torch.compile(call, fullgraph=True, backend="aot_eager")):
            loss, other, metrics, rewards = traced(case["log_probs"])
            assert loss.requires_grad and other.requires_grad and not metrics.requires_grad and not rewards.requires_grad
            assert metrics.cpu().numpy().shape == (5,) and rewards.cpu().numpy().shape == (8,)
    finally:
        torch._dynamo.reset()
