"""Operators of token models on the xdna device: the embedding, layer norm, the linear layer, linear
attention with a decay for each head, the gated feed-forward block, distillation from a teacher's top
logits, and log probabilities of given tokens.

Each is one autograd node over the gfx950 kernels (csrc/embed.hip, layer_norm.hip, gated.hip,
decay.hip, vocab.hip); the reference has no counterpart beyond its zero-copy CPU fallback
(torch_xdna_device.cpp:5124-5260).  Operands are xdna tensors; nothing falls back: a device,
dtype or shape that the kernels do not take raises, and ``set_npu_mode`` does not concern them.
Token indices are int64 or int32.  Ids and masks are data on the device and are never read by the
host, so every function can be captured in a graph; what an invalid index does is stated with each
function.  Sums and softmax statistics are fp32 and have a fixed order: equal inputs give equal
bits.  The gradients cannot be differentiated again, and an operand with a tangent (forward-mode
differentiation) raises.

    ids -> embed -> blocks -> layer_norm -> head (mm) -> distill_loss / token_log_probs
    block: layer_norm -> linear -> decay_attention -> linear (residual) -> add_layer_norm -> gated_mlp
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import device as _dev

_ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}
_LINEAR_ACTIVATIONS = {**_ACTIVATIONS, "none": 3}
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


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (biased variance):
    ``x`` [..., width] in bf16 or fp32 of any row stride, ``weight`` and ``bias`` [width] in fp32 or
    ``x``'s type.  fp32 between the loads and one rounding; the gradients of ``weight`` and ``bias``
    are fp32 sums over the rows in a fixed order."""
    return _dev.native().token_layer_norm(x, None, weight, bias, eps)[0]


class AddLayerNorm(NamedTuple):
    norm: torch.Tensor  # the norm of the sum
    sum: torch.Tensor   # x + residual


def add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   eps: float = 1e-5) -> AddLayerNorm:
    """The sum ``x + residual`` (rounded to their type) and its layer norm, in one pass: the bits of
    ``s = x + residual; layer_norm(s, weight, bias, eps)``.  Both results have gradients."""
    return AddLayerNorm(*_dev.native().token_layer_norm(x, residual, weight, bias, eps))


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "none",
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual`` in one kernel: ``x`` [..., K], ``weight`` [N, K],
    ``bias`` [N], ``residual`` [..., N], all bf16 (rows of any stride); ``activation`` "none",
    "silu", "gelu" (with erf) or "relu".  fp32 from the product to the one rounding.  For the backward
    the activation's slopes are kept in 16 bits (11 of mantissa), ReLU's as bits: its gradient is 0 where
    a unit is off, whatever comes in, and passes a NaN, as ``torch.relu``'s.  The gradient before the
    activation is rounded to bf16 for its products with ``weight`` and ``x`` (the error of theirs is 1.4
    times that of one rounding with "silu" and "gelu"; with "relu" and "none" it is exact); ``bias``'s is
    summed before that rounding."""
    return _dev.native().token_linear(x, weight, bias, residual, _choice(_LINEAR_ACTIVATIONS, activation, "activation"))


class DecayAttention(NamedTuple):
    out: torch.Tensor    # [batch, tokens, heads, dv] bf16
    state: torch.Tensor  # [batch, heads, dk, dv] fp32


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor | None = None,
                    lengths: torch.Tensor | None = None, scale: float | None = None) -> DecayAttention:
    """Causal linear attention with a decay for each head:
    ``S_t = exp(log_decay) S_{t-1} + k_t^T v_t``, ``out_t = scale q_t S_t``, for prompts and training.

    ``q`` [batch, tokens, heads, dk], ``k`` [batch, tokens, kv heads, dk], ``v`` [batch, tokens, kv heads,
    dv] in bf16, heads of 1 to 128, any strides (slices of one projection are not copied); kv heads
    divide the heads, head ``h`` of ``q`` goes with head ``h // (heads / kv heads)`` of them.  ``log_decay``
    [heads] fp32, at most 0 (``-inf``: nothing is remembered), a constant.  ``state`` [batch, heads, dk, dv]
    fp32 is the state before the first token (default: zeros); the returned one is the state behind the
    last, for the next part of the sequence or ``decay_attention_step``.  ``lengths`` [batch], taken into 0 ..
    tokens: what lies behind a sequence's end is not read, its ``out`` and gradients are 0.  ``scale`` defaults
    to ``dk ** -0.5``.

    The state is fp32; where ``q`` multiplies it, it is rounded to bf16 (at most as large an error as that of
    ``out``'s own rounding); the weighted scores have 16 bits.  ``q``, ``k``, ``v`` and ``state`` have
    gradients; those of shared heads are summed in fp32 before their one rounding.  A token whose ``k`` or
    ``v`` is not finite makes its own and the later outputs of its sequence so, and may make those of up to 63 tokens
    before it NaN (chunks of 64 tokens are multiplied whole, the later tokens with weights of 0); the gradient of ``q`` likewise.
    A ``q`` or gradient of ``out`` that is not finite makes the gradients of ``k`` and ``v`` of its own and the earlier tokens
    so, and may make those of up to 63 tokens behind it NaN."""
    return DecayAttention(*_dev.native().token_decay(q, k, v, log_decay, state, lengths, _scale(q, scale)))


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                         slots: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """One token of each sequence: updates ``state`` in place and returns ``out`` [batch, heads, dv].
    ``q`` [batch, heads, dk], ``k`` and ``v`` [batch, kv heads, size] in bf16; ``state`` [slots, heads, dk,
    dv] fp32, contiguous.  ``slots`` [batch] names each sequence's state in a pool (default: its own
    place): a negative one is an empty place of the batch (``out`` 0), one past the pool, or one that an
    earlier place of the batch has, gives NaN; none of these touches a state.  All arithmetic is fp32.
    It has no gradient and raises where one would be recorded."""
    return _dev.native().token_decay_step(q, k, v, log_decay, state, slots, _scale(q, scale))


def _scale(q: torch.Tensor, scale: float | None) -> float:
    return scale if scale is not None else max(1, q.shape[-1]) ** -0.5
