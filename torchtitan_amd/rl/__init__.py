"""Policy-gradient and preference losses around the model (the caller side of the MXFP8 linear path in RL training)."""
from .loss import (POLICY_METRICS, compute_policy_gradient_loss, compute_token_log_probs, policy_loss, preference_loss,
                   token_log_probs)

__all__ = ["POLICY_METRICS", "compute_policy_gradient_loss", "compute_token_log_probs", "policy_loss", "preference_loss",
           "token_log_probs"]
