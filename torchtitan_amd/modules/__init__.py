"""The modules whose weights the MXFP8 converter wraps (host-side mirrors of the reference's), and what runs around them."""
from .embedding import Embedding, scaled_embedding
from .linear import Linear
from .norm import ResidualRMSNorm, residual_rms_norm
from .feed_forward import FeedForward, compute_ffn_hidden_dim
from .moe import GroupedExperts, MoE, TokenChoiceTopKRouter, TokenReorderer

__all__ = ["Embedding", "scaled_embedding", "ResidualRMSNorm", "residual_rms_norm", "Linear", "FeedForward", "compute_ffn_hidden_dim", "GroupedExperts", "MoE",
           "TokenChoiceTopKRouter", "TokenReorderer"]
