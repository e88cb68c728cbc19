"""The LM head in training and in 4 bits.

* ``lm_head_cross_entropy``: softmax cross entropy over the vocabulary without
  the logits, differentiable.  The reference stops at the corruption that makes
  the labels (``csrc/ops.cpp:292-444`` of fwerkor/cid-engine v1.1.0); the loss
  over them is the step that follows.  The operators and their
  autograd formula are registered by ``_C``.
* ``QuantizedLMHead`` and the operators on it: the head's weight as 4-bit codes
  with a scale for each group of columns, its logits, and the display
  statistics over them (``csrc/ops.cpp:446-474`` takes materialised logits).
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor


def lm_head_cross_entropy(
    labels: Tensor,
    hidden: Tensor,
    weight: Tensor,
    *,
    ignore_index: int = -100,
) -> tuple[Tensor, Tensor]:
    """Per-position cross entropy of ``labels`` over ``hidden @ weight.T``
    and the positions' log-sum-exp, both float32 of the labels' shape, without
    writing the ``[*, vocab]`` logits.

    ``hidden [*labels.shape, H]`` and ``weight [vocab, H]`` are both bfloat16
    or both float16, H a multiple of 8.  A position whose label is
    ``ignore_index`` (what ``display_corrupt_from_random`` writes where there
    is no loss) has both outputs 0, its hidden state is not read, and its
    gradient is 0.  Any other label outside ``[0, vocab)`` gives NaN outputs
    and a NaN gradient of that position, takes no part in the weight's
    gradient and sets ``STATUS_TOKEN_ID_OUT_OF_RANGE``.

    Differentiable once in ``hidden`` and ``weight``, through both outputs:
    weight the positions (``(loss * scale).sum()``), average them, or add a
    penalty of the log-sum-exp.  Inputs with a forward-mode tangent (dual
    tensors, ``torch.func.jvp``) are refused.  The backward computes the logits
    again, a piece of the vocabulary at a time, and holds their gradient in the
    inputs' dtype; in float16 it is scaled by one power of two, so that elements
    below 2^-37 of the largest position weight are lost."""
    return torch.ops.cid_engine.lm_head_cross_entropy(labels, hidden, weight, ignore_index)


class QuantizedLMHead(NamedTuple):
    """A ``[vocab, H]`` weight in 4 bits, as ``lm_head_quantize`` lays it out:
    ``packed`` int32 ``[vocab, H / 8]`` (codes q in [-8, 7], stored as q + 8;
    column 8 j + 2 i at bits 4 i of word j, column 8 j + 2 i + 1 at bits
    16 + 4 i) and ``scales`` ``[vocab, H / group]``, standing for scale * q.
    ``refine_step_from_hidden`` and ``DisplayRefineLoop`` take it in place of
    the bfloat16 weight."""

    packed: Tensor
    scales: Tensor


def lm_head_quantize(weight: Tensor, *, group_size: int = 128) -> QuantizedLMHead:
    """The 4-bit form of a bfloat16 or float16 ``[vocab, H]`` weight: for each
    group of ``group_size`` (32, 64 or 128) columns, scale = max |w| / 7 in the
    weight's dtype and codes w / scale rounded to nearest (ties to even).  A
    group of zeros has scale 0; a group with a NaN or infinite weight has that
    scale and codes 0."""
    return QuantizedLMHead(*torch.ops.cid_engine.lm_head_quantize(weight, group_size))


def lm_head_dequantize(packed: Tensor, scales: Tensor) -> Tensor:
    """The weight that codes and scales stand for, rounded to the scales'
    dtype."""
    return torch.ops.cid_engine.lm_head_dequantize(packed, scales)


def lm_head_quantized_logits(hidden: Tensor, packed: Tensor, scales: Tensor) -> Tensor:
    """``hidden [*, H]`` times the 4-bit weight: ``[*, vocab]`` logits in
    hidden's dtype (the scales' dtype too).  Each group's sum is accumulated
    and scaled in float32; the logits are rounded once.  Made for few rows:
    the weight is read once for every 64 of them (32 with groups of 64, 16
    with groups of 32), and beyond that the 16-bit weight is faster.  H is at most 32768.  A hidden row with
    a NaN or infinite value has NaN logits, and so has a column with a NaN or
    infinite scale.  Not differentiable."""
    return torch.ops.cid_engine.lm_head_quantized_logits(hidden, packed, scales)


def lm_head_quantized_display_statistics(
    token_ids: Tensor,
    hidden: Tensor,
    packed: Tensor,
    scales: Tensor,
    *,
    round_bf16: bool = True,
) -> tuple[Tensor, Tensor, Tensor]:
    """``display_token_statistics`` over the 4-bit head's float32 logits, each
    rounded to bfloat16 first when ``round_bf16`` (as
    ``lm_head_display_statistics``), without writing them."""
    return torch.ops.cid_engine.lm_head_quantized_display_statistics(token_ids, hidden, packed,
                                                                     scales, round_bf16)
