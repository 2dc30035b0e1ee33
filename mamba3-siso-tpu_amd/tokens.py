"""The two ends of the language model as differentiable operators: the embedding lookup that
turns tokens into rows, and what is read off the logits (`token_logprobs`, `distill_loss`).

Each is one autograd node over the HIP kernels of ``csrc/m3s_embed.hip`` and
``csrc/m3s_vocab.hip``, or a plain launch where no gradient is taken. The nodes have no
forward-mode rule and are differentiable once. The lookup's is in C++ (``csrc/m3s_nodes.cpp``).
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import kernels as K
from . import layer as LY

Tensor = torch.Tensor


def _needs_node(*tensors) -> bool:
    """Whether a call goes through its autograd node: a gradient is taken, or the node has to
    refuse what a bare launch would drop (a forward-mode tangent) or record wrongly (a trace)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                return True
    return torch.jit.is_tracing() or LY.has_tangent(*tensors)


class _EmbedFn(torch.autograd.Function):
    """`kernels.embedding_forward` / `kernels.embedding_backward` as a node in Python, for what the
    one in C++ does not take: strided ids or columns, a trace, and a tangent, which it refuses."""

    @staticmethod
    def forward(ctx, table, tokens, scale, padding_idx):
        tokens = tokens.contiguous()
        y = K.embedding_forward(table, tokens, scale)
        ctx.save_for_backward(tokens)
        ctx.call = table.shape[0], scale, padding_idx if padding_idx >= 0 else None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (tokens,) = ctx.saved_tensors
        return K.embedding_backward(tokens, dy, *ctx.call), None, None, None


def embed_tokens(table: Tensor, tokens: Tensor, scale: float = 1.0,
                 padding_idx: Optional[int] = None) -> Tensor:
    """``scale * table[tokens]``, differentiable in ``table`` (V, D) float32 or bf16; ``tokens``
    int32 or int64 of any shape, on the table's device.

    The gradient is dense, summed in float32 in a fixed order and so bit-reproducible.
    ``padding_idx`` names an id (negative: from the end) whose row is looked up but gets no
    gradient. An id outside [0, V) gives a row of NaN, and no gradient."""
    if table.dim() != 2:
        raise ValueError(f"embedding: the table must be (V, D), got {tuple(table.shape)}")
    pad = -1 if padding_idx is None else K.embedding_padding(int(padding_idx), table.shape[0])
    y = _lib.nodes().embed(table, tokens, scale, pad, K.POISON_OUTPUTS)
    if y is not None:
        return y
    if _needs_node(table):
        return _EmbedFn.apply(table, tokens, float(scale), pad)
    return K.embedding_forward(table, tokens, scale)


class TokenLogprobs(NamedTuple):
    """`token_logprobs`' results; see there. ``logp`` is None without targets, ``top_logp`` and
    ``top_ids`` without ``top``."""

    logp: Optional[Tensor]
    entropy: Tensor
    top_logp: Optional[Tensor]
    top_ids: Optional[Tensor]


class _LogprobFn(torch.autograd.Function):
    """`kernels.logprob_forward` / `kernels.logprob_backward` as one node."""

    @staticmethod
    def forward(ctx, logits, targets, top, temperature, ignore_index):
        out, targets, ctx.call = K.logprob_call(logits, targets, top, temperature, ignore_index)
        logp, entropy, top_logp, top_ids, stats = out
        ctx.save_for_backward(logits, targets, stats, top_ids)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if top_ids is not None:
            ctx.mark_non_differentiable(top_ids)
        return logp, entropy, top_logp, top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dentropy, dtop_logp, _):
        if dlogp is None and dentropy is None and dtop_logp is None:
            return None, None, None, None, None
        saved = logits, targets, stats, top_ids = ctx.saved_tensors
        a = ctx.call.again(saved)
        if a is not None:
            dx = K.logprob_call_backward(a, ctx.call.device, logits, dlogp, dentropy, dtop_logp)
        else:
            dx = K.logprob_backward(logits, targets, stats, top_ids, dlogp, dentropy, dtop_logp,
                                    ctx.temperature, ctx.call.args.ignore_index)
        return dx, None, None, None, None


def token_logprobs(logits: Tensor, targets: Optional[Tensor] = None, top: int = 0,
                   temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """What a row of ``logits`` (..., V), float32 or bf16, says about tokens: `TokenLogprobs` of
    float32 ``logp`` (...,), ``log softmax(logits / temperature)`` at ``targets`` (...,);
    ``entropy`` (...,) of that distribution; ``top_logp`` and int64 ``top_ids`` (..., top), its
    ``top`` (at most 64) best ids in falling order, of equal logits the lower id first.

    ``logp``, ``entropy`` and ``top_logp`` are differentiable in ``logits``. ``logits`` may be a
    strided view (``logits[:, :-1]`` against ``tokens[:, 1:]`` makes no copy). Positions whose
    target is ``ignore_index`` are padding: their logits are not read, logp and entropy are 0, ids
    -1 (which `distill_loss` takes for no entry) and their gradient is 0. Any other target outside
    [0, V) gives NaN; a row of nothing but -inf has logp -inf, entropy 0 and no gradient; a row with
    a NaN or +inf is NaN, with ids -1."""
    if _needs_node(logits):
        return TokenLogprobs(*_LogprobFn.apply(logits, targets, int(top), float(temperature),
                                               int(ignore_index)))
    return TokenLogprobs(*K.logprob_call(logits, targets, int(top), temperature, int(ignore_index), False)[0][:4])


class DistillLoss(NamedTuple):
    """`distill_loss`' per-row results; ``nll`` is None without targets."""

    kd: Tensor
    nll: Optional[Tensor]


class _DistillFn(torch.autograd.Function):
    """`kernels.distill_forward` / `kernels.distill_backward` as one node."""

    @staticmethod
    def forward(ctx, logits, ids, teacher, targets, temperature, ignore_index):
        (kd, nll, stats), ops, ctx.call = K.distill_call(logits, ids, teacher, targets, temperature,
                                                         ignore_index)
        ctx.save_for_backward(logits, *ops, stats)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        return kd, nll

    @staticmethod
    @once_differentiable
    def backward(ctx, dkd, dnll):
        if dkd is None and dnll is None:
            return None, None, None, None, None, None
        saved = logits, ids, teacher, targets, stats = ctx.saved_tensors
        a = ctx.call.again(saved)
        if a is not None:
            dx = K.distill_call_backward(a, ctx.call.device, logits, dkd, dnll)
        else:
            dx = K.distill_backward(logits, ids, teacher, targets, stats, dkd, dnll, ctx.temperature,
                                    ctx.call.args.ignore_index)
        return dx, None, None, None, None, None


def distill_loss(logits: Tensor, teacher_ids: Tensor, teacher_logits: Tensor,
                 temperature: float = 1.0, targets: Optional[Tensor] = None,
                 ignore_index: int = -100) -> DistillLoss:
    """The loss of a student's ``logits`` (..., V) against a teacher's best K (at most 256) tokens,
    per row in float32, differentiable in ``logits``: `DistillLoss` of ``kd = T^2 sum_i w_i (log w_i
    - log softmax(logits / T)[id_i])`` with ``w = softmax(teacher_logits / T)`` over the K entries
    (log-probabilities as `token_logprobs` gives them serve as well), and with ``targets``
    ``nll = -log softmax(logits)[target]``, the cross-entropy, from the same pass.

    Entries with an id < 0 do not count; a row without any has kd 0, one whose target is
    ``ignore_index`` nll 0, and neither sends a gradient (nor is a row without both read). A
    repeated id adds up. An id >= V, or another target outside [0, V), gives NaN. The teacher is a
    constant: logits of it that require a gradient are refused."""
    if torch.is_grad_enabled() and teacher_logits.requires_grad:
        raise ValueError("distill_loss: the teacher's logits must not require a gradient (detach them)")
    if _needs_node(logits, teacher_logits):
        return DistillLoss(*_DistillFn.apply(logits, teacher_ids, teacher_logits, targets,
                                             float(temperature), int(ignore_index)))
    return DistillLoss(*K.distill_call(logits, teacher_ids, teacher_logits, targets, temperature,
                                       int(ignore_index), False)[0][:2])
