"""The two ends of the language model as differentiable operators: the embedding lookup that
turns tokens into rows, and what is read off the logits (`token_logprobs`, `distill_loss`).

Each is one autograd node over the HIP kernels of ``csrc/m3s_embed.hip`` and
``csrc/m3s_vocab.hip``, or a plain launch where no gradient is taken. The nodes have no
forward-mode rule and are differentiable once.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import kernels as K
from . import layer as LY

Tensor = torch.Tensor


def _needs_node(*tensors) -> bool:
    """Whether a call goes through its autograd node: a gradient is taken, or the node has to
    refuse what a bare launch would drop (a forward-mode tangent) or record wrongly (a trace)."""
    return ((torch.is_grad_enabled() and any(t.requires_grad for t in tensors))
            or torch.jit.is_tracing() or LY.has_tangent(*tensors))


class _EmbedFn(torch.autograd.Function):
    """`kernels.embedding_forward` / `kernels.embedding_backward` as one node."""

    @staticmethod
    def forward(ctx, table, tokens, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.vocab, ctx.scale, ctx.padding_idx = table.shape[0], scale, padding_idx
        return K.embedding_forward(table, tokens, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (tokens,) = ctx.saved_tensors
        return K.embedding_backward(tokens, dy, ctx.vocab, ctx.scale, ctx.padding_idx), None, None, None


def embed_tokens(table: Tensor, tokens: Tensor, scale: float = 1.0,
                 padding_idx: Optional[int] = None) -> Tensor:
    """``scale * table[tokens]``, differentiable in ``table`` (V, D) float32 or bf16; ``tokens``
    int32 or int64 of any shape, on the table's device.

    The gradient is dense, summed in float32 in position order and so bit-reproducible.
    ``padding_idx`` names an id (negative: from the end) whose row is looked up but gets no
    gradient. An id outside [0, V) gives a row of NaN, and no gradient."""
    if padding_idx is not None:
        padding_idx = K.embedding_padding(int(padding_idx), table.shape[0])
    if _needs_node(table):
        return _EmbedFn.apply(table, tokens, float(scale), padding_idx)
    return K.embedding_forward(table, tokens, scale)
