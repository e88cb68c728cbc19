"""The LM head in training: softmax cross entropy over the vocabulary without
the logits, differentiable.

The reference stops at the corruption that makes the labels
(``csrc/ops.cpp:292-444`` of fwerkor/cid-engine v1.1.0); the loss over them is
the step that follows.  The operators are registered by ``_C``; this module
registers their autograd formula.
"""

from __future__ import annotations

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
    penalty of the log-sum-exp.  The backward computes the logits again, a
    piece of the vocabulary at a time."""
    return torch.ops.cid_engine.lm_head_cross_entropy(labels, hidden, weight, ignore_index)


def _setup(ctx, inputs, output) -> None:
    labels, hidden, weight, ignore_index = inputs
    ctx.ignore_index = ignore_index
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(labels, hidden, weight, output[1])


def _backward(ctx, grad_loss, grad_lse):
    labels, hidden, weight, lse = ctx.saved_tensors
    need_hidden, need_weight = ctx.needs_input_grad[1:3]
    if grad_loss is None and grad_lse is None:
        return None, None, None, None
    gh, gw = torch.ops.cid_engine.lm_head_cross_entropy_backward(
        grad_loss, grad_lse, labels, hidden, weight, lse, ctx.ignore_index,
        need_hidden, need_weight)
    return None, gh if need_hidden else None, gw if need_weight else None, None


def _no_second_backward(ctx, *grads):
    raise RuntimeError("cid_engine.lm_head_cross_entropy is differentiable once: "
                       "its gradient has no gradient")


torch.library.register_autograd("cid_engine::lm_head_cross_entropy", _backward,
                                setup_context=_setup)
torch.library.register_autograd("cid_engine::lm_head_cross_entropy_backward",
                                _no_second_backward)
