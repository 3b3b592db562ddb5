"""Operators of token models on the xdna device: the embedding, the gated feed-forward block,
distillation from a teacher's top logits, and log probabilities of given tokens.

Each is one autograd node over the gfx950 kernels (csrc/embed.hip, gated.hip, vocab.hip); the
reference has no counterpart beyond its zero-copy CPU fallback
(torch_xdna_device.cpp:5124-5260).  Operands are xdna tensors; nothing falls back: a device,
dtype or shape that the kernels do not take raises, and ``set_npu_mode`` does not concern them.
Token indices are int64 or int32.  Ids and masks are data on the device and are never read by the
host, so every function can be captured in a graph; what an invalid index does is stated with each
function.  Sums and softmax statistics are fp32 and have a fixed order: equal inputs give equal
bits.  The gradients cannot be differentiated again, and an operand with a tangent (forward-mode
differentiation) raises.

    ids -> embed -> gated_mlp -> head (mm) -> distill_loss / token_log_probs
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import device as _dev

_ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _choice(table: dict, value: str, what: str) -> int:
    try:
        return table[value]
    except (KeyError, TypeError):
        raise ValueError(f"{what} must be one of {', '.join(table)}, got {value!r}") from None


def embed(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[ids]``: ``ids`` of any shape, ``weight`` [tokens, width] in bf16 or fp32
    (any row stride), each element rounded once.

    The gradient of ``weight`` is dense: per row the fp32 sum of its tokens' gradients in token
    order, times ``scale``, rounded once.  ``padding_idx`` rows get none.  An id outside the
    table looks up a row of NaN and has no gradient."""
    return _dev.native().token_embed(ids, weight, scale, padding_idx)


def gated_linear(x: torch.Tensor, w_in: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """``act(x @ w_in[:F].T) * (x @ w_in[F:].T)`` in one kernel: ``x`` [..., K], ``w_in``
    [2 F, K] (gate rows, then up rows), both bf16; ``activation`` "silu", "gelu" (with erf) or
    "relu".  The projections stay in fp32 through the activation and the product; for the
    backward they are kept in 20 bits each."""
    return _dev.native().token_gated_linear(x, w_in, _choice(_ACTIVATIONS, activation, "activation"))


def gated_mlp(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """The gated feed-forward block, ``gated_linear(x, w_in, activation) @ w_out.T``, ``w_out``
    [N, F] bf16, as one autograd node."""
    return _dev.native().token_gated_mlp(x, w_in, w_out, _choice(_ACTIVATIONS, activation, "activation"))


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, temperature: float = 1.0,
                 weight: torch.Tensor | None = None, reduction: str = "mean") -> torch.Tensor:
    """Distillation from a teacher's top logits: per row, with ``p`` the softmax of
    ``teacher_logits / temperature`` over the row's entries and ``q`` the softmax of
    ``logits / temperature`` over the vocabulary, ``temperature**2 * sum p (ln p - ln q)``.

    ``logits`` [..., vocabulary] in bf16 or fp32; ``teacher_ids`` and ``teacher_logits`` [..., k],
    k up to 1024.  An entry with a negative id or a logit of -inf is absent.  The sum goes over the
    entries: a token named twice is two terms with a ``p`` each, which differs from the divergence
    of the joined entries by a constant, not in its gradient (``q`` minus their sum).  The id of an
    entry that is present past the vocabulary makes the row's loss NaN and leaves the row out of
    the gradient.  ``weight`` [...] scales rows (0: the row is left out, whatever it holds); a row without
    entries has weight 0.  ``reduction`` "mean" divides by the sum of the weights (0 where that
    is 0), "sum" does not, "none" gives the weighted row losses.  The loss is fp32; the gradient
    goes to ``logits`` only."""
    return _dev.native().token_distill(logits, teacher_ids, teacher_logits, temperature, weight,
                                       _choice(_REDUCTIONS, reduction, "reduction"))


class TokenLogProbs(NamedTuple):
    log_probs: torch.Tensor      # [...] fp32
    entropy: torch.Tensor        # [...] fp32
    top_log_probs: torch.Tensor  # [..., top_k] fp32, no gradient
    top_ids: torch.Tensor        # [..., top_k] int64


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor, top_k: int = 0, temperature: float = 1.0) -> TokenLogProbs:
    """Log probabilities of ``targets`` [...] under ``softmax(logits / temperature)``, the
    distribution's entropy, and its ``top_k`` (up to 64) most likely tokens, ties to the lowest
    index.  ``logits`` [..., vocabulary] in bf16 or fp32; masked tokens are -inf.

    ``log_probs`` and ``entropy`` have a gradient in ``logits``.  A negative target is not
    scored (0, no gradient), one past the vocabulary gives NaN (and no gradient).  A masked token's
    gradient is 0, unless it is the target: that has the derivative of its own logit, 1 /
    ``temperature``, beside a log probability of -inf.  A row of -inf only has log probabilities of
    -inf, entropy 0 and no gradient."""
    return TokenLogProbs(*_dev.native().token_log_probs(logits, targets, top_k, temperature))
