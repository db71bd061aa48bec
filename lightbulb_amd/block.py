"""A decoder layer: attention and MLP on a residual stream, with the norms between them.

``CustomTransformerBlock`` of the reference (src/model/custom_transformer_block.rs:329: input norm, attention,
residual, post-attention norm, MLP, residual), and the forms of it that also norm a block's output, gate it or
scale it into the stream.  What stands between two products is one ``int8.residual_norm`` call: the stream's
update, the next norm and, where the products behind it are 8-bit integer ones, their codes.
"""
from __future__ import annotations

import torch

from .attention import Attention, KvCache, Step
from .int8 import Int8Tokens, Norm, residual_norm
from .quantized import Mlp


class Block:
    """``h = x + scale * attn_gate * attn_post(attention(input_norm(x)))``, then
    ``y = h + scale * mlp_gate * mlp_post(mlp(mlp_norm(h)))``.

    The post norms and the gates (one value a channel, of the stream's type) may be None."""

    def __init__(self, attention: Attention, mlp: Mlp, input_norm: Norm, mlp_norm: Norm, *, attn_post: Norm | None = None,
                 mlp_post: Norm | None = None, attn_gate: torch.Tensor | None = None, mlp_gate: torch.Tensor | None = None, scale: float = 1.0):
        self.attention, self.mlp = attention, mlp
        self.input_norm, self.mlp_norm, self.attn_post, self.mlp_post = input_norm, mlp_norm, attn_post, mlp_post
        self.attn_gate, self.mlp_gate, self.scale = attn_gate, mlp_gate, scale

    # codes straight from the norm where every product behind it takes them
    def _attn_codes(self) -> bool:
        a = self.attention
        return a.q_proj.is_int8() and a.k_proj.is_int8() and a.v_proj.is_int8()

    def _mlp_codes(self) -> bool:
        return self.mlp.gate_proj.is_int8() and self.mlp.up_proj.is_int8()

    def normed(self, xs: torch.Tensor) -> "torch.Tensor | Int8Tokens":
        """``input_norm(xs)`` as the attention takes it."""
        return residual_norm(xs, norm=self.input_norm, quantize=self._attn_codes())[1]

    def forward(self, xs: torch.Tensor, cache: KvCache, step: Step, normed: "torch.Tensor | Int8Tokens | None" = None,
                next: "Block | None" = None) -> tuple[torch.Tensor, "torch.Tensor | Int8Tokens | None"]:
        """The stream ``xs`` [step.num_tokens, hidden] behind the block and, given the block after it, what that takes
        as ``normed``: its norm is formed with this block's last update.  ``normed`` None: the input norm is formed
        here.  Rows behind the last sequence's come out unset."""
        a = self.attention(self.normed(xs) if normed is None else normed, cache, step)
        h, b = residual_norm(a, xs, post=self.attn_post, gate=self.attn_gate, scale=self.scale, norm=self.mlp_norm, quantize=self._mlp_codes())
        y = self.mlp(b)
        after, codes = (None, False) if next is None else (next.input_norm, next._attn_codes())
        return residual_norm(y, h, post=self.mlp_post, gate=self.mlp_gate, scale=self.scale, norm=after, quantize=codes)

    __call__ = forward
