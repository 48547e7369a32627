"""CPU: the losses' edges in torch operations."""
import pytest

from tests import sequence_loss_edges as edges


@pytest.mark.parametrize("case", ["a_rejected_answer_without_a_chance", "a_token_that_the_reference_rules_out",
                                  "as_many_tokens_as_sequences", "a_border_between_two_float32_numbers", "operands_from_inference_mode"])
def test_edge(case):
    getattr(edges, case)("cpu")
