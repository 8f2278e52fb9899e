"""The choice of tokens for a batch (next to the reference's softmax_sample,
src/kernels/shaders.zig:826-887)."""
from __future__ import annotations

from .. import ops


class SampleTokens:
    """tokens[row] (i32) of each row of logits by its temperature, top_k (i32), top_p and min_p, each a
    buffer of rows or None, and its random number in [0, 1); kept[row] (i32 or None) = tokens that the
    filters leave."""

    def __init__(self, device):
        self.device = device

    @classmethod
    def init(cls, device) -> "SampleTokens":
        return cls(device)

    def forward(self, logits, temperature, top_k, top_p, min_p, random, tokens, kept=None, dtype="f32"):
        rows = tokens.count
        ops.sample_tokens(self.device, logits, temperature, top_k, top_p, min_p, random, tokens, kept,
                          rows, logits.count // rows, dtype)
