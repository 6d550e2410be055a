"""Operators on rows of output logits, next to the transducer losses: log-probs of given tokens with the entropy and the
most likely alternatives (what a decoder, a rescoring pass or a teacher's labelling asks of a model), and distillation
from a teacher's listed log-probs, on any batch of rows and on the pruned lattice of ``rnnt_loss_pruned``.

No counterpart in the reference.  Each is one fused HIP kernel forward and one backward (k2_amd/csrc/token_logprobs.hip,
k2_amd/csrc/distillation.hip) behind a torch.autograd.Function.  Logits are float32, float16 or bfloat16 device tensors,
[..., C], any strides; sums and results are float32, gradients have the logits' type.  There are no second derivatives, and no
forward-mode ones: a tensor that carries a tangent is refused (NotImplementedError).
"""
import math
from typing import NamedTuple, Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import native
from .rnnt_loss import _dev_i64

RESTS = ("renormalise", "bucket")


class TokenLogprobs(NamedTuple):
    """What ``get_token_logprobs`` returns; what was not asked for is None."""
    logprobs: Optional[Tensor]
    entropy: Optional[Tensor]
    top_logprobs: Optional[Tensor]
    top_tokens: Optional[Tensor]


class _TokenLogprobs(torch.autograd.Function):
    """The node of the ctypes host; the extension has its own (csrc/pybind.cpp)."""

    @staticmethod
    def forward(ctx, logits, tokens, mask, temperature, num_top, return_entropy):
        logprobs, entropy, top_logprobs, top_tokens, stats = native.token_logprobs_forward(
            logits, tokens, mask, temperature, num_top, return_entropy, ctx.needs_input_grad[0])
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, tokens, mask, stats, entropy, top_tokens)
        ctx.temperature = temperature
        if top_tokens is not None:
            ctx.mark_non_differentiable(top_tokens)
        return logprobs, entropy, top_logprobs, top_tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, logprobs_grad, entropy_grad, top_grad, _):
        if logprobs_grad is None and entropy_grad is None and top_grad is None:
            return (None,) * 6
        logits, tokens, mask, stats, entropy, top_tokens = ctx.saved_tensors
        grad = native.token_logprobs_backward(logits, tokens, mask, stats, entropy, top_tokens, _dense(logprobs_grad),
                                              _dense(entropy_grad), _dense(top_grad), ctx.temperature)
        return grad, None, None, None, None, None


class _Distillation(torch.autograd.Function):
    """The node of the ctypes host, as above.  The loss of each row, or sums of them: ``sums`` -1 leaves the rows, n >= 0
    makes n sums of equally many rows each.  ``mean``: divided by the number of rows that count.  ``factor`` multiplies the sums."""

    @staticmethod
    def forward(ctx, logits, top_logprobs, top_tokens, mask, temperature, bucket, sums, mean, factor):
        rows, records = native.distillation_forward(logits, top_logprobs, top_tokens, mask, temperature, bucket,
                                                    ctx.needs_input_grad[0])
        loss, inverse_count = (rows, None) if sums < 0 else native.distillation_sum(rows, mask, sums, mean, factor)
        if records is not None:
            ctx.save_for_backward(logits, top_logprobs, top_tokens, records, inverse_count if mean else None)
            ctx.meta = (temperature, bucket, factor)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, loss_grad):
        logits, top_logprobs, top_tokens, records, inverse_count = ctx.saved_tensors
        temperature, bucket, factor = ctx.meta
        grad = native.distillation_backward(logits, top_logprobs, top_tokens, records, _dense(loss_grad), inverse_count,
                                            factor, temperature, bucket)
        return (grad,) + (None,) * 8


def _dense(t: Optional[Tensor]) -> Optional[Tensor]:
    return None if t is None else t.resolve_neg().contiguous()


def _check_logits(logits: Tensor, mask: Optional[Tensor], temperature: float) -> Optional[Tensor]:
    """The checks all operators share; the mask as the host layers take it."""
    assert logits.ndim >= 1, logits.shape
    assert logits.shape[-1] >= 1, logits.shape
    assert temperature > 0.0 and math.isfinite(temperature), temperature
    if mask is None:
        return None
    assert mask.dtype == torch.bool, mask.dtype
    assert mask.shape == logits.shape[:-1], (mask.shape, logits.shape)
    return mask.to(logits.device).contiguous()


def get_token_logprobs(
    logits: Tensor,
    tokens: Optional[Tensor] = None,
    mask: Optional[Tensor] = None,
    temperature: float = 1.0,
    num_top: int = 0,
    return_entropy: bool = False,
) -> TokenLogprobs:
    """Log-probs under softmax(logits / temperature), one pass over the logits.

    Args:
      logits: [..., C].
      tokens: int64, the shape of the rows ([...]: one token a row) or [..., n] with n <= 64.  A negative token (padding)
        has log-prob 0 and adds nothing to the gradient; one of C and above is a mistake and gives NaN.
      mask: bool [...]; rows with False do not count, whatever they hold: log-prob 0, entropy 0, no alternatives, gradient 0.
      temperature: positive; it and log2(e) / temperature have to be float32 numbers.
      num_top: how many alternatives to list, at most 64: the largest logits of each row in falling order, the lower index
        first where two are equal.
      return_entropy: whether to return the entropy of each row.

    Returns:
      (logprobs, entropy, top_logprobs, top_tokens): float32 of tokens' shape, float32 [...], float32 [..., num_top] and
      int64 [..., num_top], each None where it was not asked for.  Past the C-th alternative and in rows masked out the
      list holds -inf and -1, which ``distillation_loss`` takes as "no entry".  Gradients flow to logits from the first
      three.  A row of nothing but -inf has log-probs -inf, entropy 0 and gradient 0."""
    mask = _check_logits(logits, mask, temperature)
    lead = logits.shape[:-1]
    if tokens is not None:
        assert tokens.shape == lead or tokens.shape[:-1] == lead, (tokens.shape, logits.shape)
        assert tokens.shape == lead or 1 <= tokens.shape[-1] <= native.MAX_TOKENS, tokens.shape
        tokens = _dev_i64(tokens, logits)
    num_top = int(num_top)
    assert 0 <= num_top <= native.MAX_TOP, num_top
    args = (logits, tokens, mask, float(temperature), num_top, bool(return_entropy))
    results = native.token_logprobs(*args)
    if results is None:
        results = _TokenLogprobs.apply(*args)
    return TokenLogprobs(*results)


def _distill(args, sums, mean, factor, scalar):
    loss = native.distillation(*args, sums, mean, factor, scalar)
    if loss is None:
        loss = _Distillation.apply(*args, sums, mean, factor)
        loss = loss.reshape(()) if scalar else loss
    return loss


def _distillation_args(logits, top_logprobs, top_tokens, mask, temperature, rest, reduction):
    mask = _check_logits(logits, mask, temperature)
    assert top_tokens.shape == top_logprobs.shape, (top_tokens.shape, top_logprobs.shape)
    assert top_tokens.shape[:-1] == logits.shape[:-1] and top_tokens.ndim == logits.ndim, (top_tokens.shape, logits.shape)
    assert 1 <= top_tokens.shape[-1] <= native.MAX_TEACHER, top_tokens.shape
    assert top_logprobs.is_floating_point(), top_logprobs.dtype
    assert not top_logprobs.requires_grad, "the teacher's log-probs are constants: pass top_logprobs.detach()"
    if rest not in RESTS:
        raise ValueError(f"rest should be ('renormalise' | 'bucket'), given {rest}")
    if reduction not in ("none", "mean", "sum"):
        raise ValueError(f"reduction should be ('none' | 'mean' | 'sum'), given {reduction}")
    return (logits, _dense(top_logprobs.to(device=logits.device, dtype=torch.float32)), _dev_i64(top_tokens, logits), mask,
            float(temperature), rest == "bucket")


def distillation_loss(
    logits: Tensor,
    top_logprobs: Tensor,
    top_tokens: Tensor,
    mask: Optional[Tensor] = None,
    temperature: float = 1.0,
    rest: str = "renormalise",
    reduction: Optional[str] = "mean",
) -> Tensor:
    """KL(teacher || student) from the teacher's most likely tokens of each row, as ``get_token_logprobs`` lists them.

    Args:
      logits: the student's, [..., C]; its distribution is softmax(logits / temperature).
      top_logprobs: [..., K] with K <= 256, the teacher's log-probs at the same temperature; no gradient flows to them.  NaN or
        +inf at a token (what a teacher row gives that overflowed its type) makes its row's loss and gradient NaN; -inf is
        probability 0.
      top_tokens: int64 [..., K]; a negative one is no entry, one of C and above is a mistake and gives NaN.  A token listed
        twice counts with both entries.
      mask: bool [...]; rows with False do not count, whatever they hold: loss 0, gradient 0.
      rest: "renormalise" scales the listed probabilities to sum to one; "bucket" leaves them as they are and compares what
        they leave of one with the student's total outside the list, as one more outcome (a row whose student has nothing
        outside the list has no such outcome).
      reduction: "none" gives the loss of each row [...], "sum" their sum, "mean" that divided by the number of rows that
        mask leaves (0 if it leaves none).  A row without any entry has loss 0.

    Gradients scale with 1 / temperature; multiply the loss by temperature ** 2 to keep them comparable across
    temperatures."""
    args = _distillation_args(logits, top_logprobs, top_tokens, mask, temperature, rest, reduction)
    if reduction == "none":
        return _distill(args, -1, False, 1.0, False)
    return _distill(args, 1, reduction == "mean", 1.0, True)


def get_pruned_mask(ranges: Tensor, boundary: Tensor) -> Tensor:
    """bool [B][T][s_range]: which rows of a pruned lattice (``ranges`` from get_rnnt_prune_ranges, int64 [B][T][s_range])
    lie inside their sequence's ``boundary`` ([B][4] int64: begin_symbol, begin_frame, end_symbol, end_frame), the rows
    that ``rnnt_loss_pruned`` can reach.  The mask for the operators above on a pruned lattice's logits."""
    assert ranges.ndim == 3, ranges.shape
    assert boundary.shape == (ranges.shape[0], 4), (boundary.shape, ranges.shape)
    return native.pruned_mask(_dev_i64(ranges, ranges), _dev_i64(boundary, ranges))


def rnnt_distillation_loss_pruned(
    logits: Tensor,
    top_logprobs: Tensor,
    top_tokens: Tensor,
    ranges: Tensor,
    boundary: Optional[Tensor] = None,
    temperature: float = 1.0,
    rest: str = "renormalise",
    reduction: Optional[str] = "mean",
) -> Tensor:
    """``distillation_loss`` on the pruned lattice, next to ``rnnt_loss_pruned`` and with its logits [B][T][s_range][C],
    ranges [B][T][s_range] and boundary: the losses of a sequence's lattice rows inside its boundary are summed, and
    ``reduction`` works on the sequences: "none" [B], "sum", or "mean" over B.  top_logprobs and top_tokens
    [B][T][s_range][K] are the teacher's on the same lattice."""
    assert logits.ndim == 4, logits.shape
    B = logits.shape[0]
    assert ranges.shape == logits.shape[:3], (ranges.shape, logits.shape)
    mask = None if boundary is None else get_pruned_mask(ranges, boundary)
    args = _distillation_args(logits, top_logprobs, top_tokens, mask, temperature, rest, reduction)
    if reduction == "none":
        return _distill(args, B, False, 1.0, False)
    return _distill(args, 1, False, 1.0 if reduction == "sum" else 1.0 / max(B, 1), True)
