"""Losses over the logits of a language-model head without an fp32 copy of the rows x vocab matrix: softmax cross-entropy for
bf16 logits (csrc/ops/cross_entropy.cu: one read of the logits in the forward pass, the gradient written in bf16 over them in
the backward pass) and the clipped policy loss with a KL term (csrc/ops/policy_loss.cu)."""
from __future__ import annotations

import torch

from .. import _ext


def launches() -> int:
    return _ext.load().launches("loss")


def fused_cross_entropy(logits: torch.Tensor, targets: torch.Tensor, vocab: int | None = None) -> torch.Tensor:
    """Mean cross-entropy of bf16 `logits` [rows, width] against int64 `targets` [rows]; columns at or beyond
    `vocab` (padding of the output projection) take no probability mass and get zero gradient."""
    if not logits.is_cuda:
        raise RuntimeError("fused_cross_entropy runs on CUDA (sm_100a) only")
    assert logits.dim() == 2 and logits.dtype == torch.bfloat16 and logits.stride(1) == 1
    assert targets.dtype == torch.int64 and targets.is_contiguous() and targets.numel() == logits.shape[0]
    loss = _ext.load().cross_entropy(logits, targets, vocab)
    if loss is None:
        raise ValueError("fused_cross_entropy: logits and targets do not fit together")
    return loss


_LOGITS = (torch.bfloat16, torch.float16, torch.float32)


def fused_policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                      ref_logp: torch.Tensor | None = None, weights: torch.Tensor | None = None, clip: tuple[float, float] = (0.2, 0.2),
                      kl_coef: float = 0.0, vocab: int | None = None, reduction: str = "mean") -> tuple[torch.Tensor, torch.Tensor]:
    """Clipped policy loss with a KL term (csrc/ops/policy_loss.cu) over `logits` [rows, width] (bf16, fp16 or fp32); returns the loss
    (fp32) and the log-probability of every row's token (fp32 [rows], a constant for autograd).

    With lp = log p(token), r = exp(lp - old_logp) and A = advantages, a row's term is
    -min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_coef (exp(ref_logp - lp) - (ref_logp - lp) - 1).  The loss is the sum of
    weights x terms, with `reduction="mean"` over the sum of the weights (zero, with a zero gradient, where that is zero).  A row of
    weight zero takes no part whatever it holds (padding); one of another weight whose token is outside the vocabulary makes the loss
    NaN.  The last KL factor needs `ref_logp`.  Per row: int64 `tokens`, fp32 `old_logp`, `advantages`, `ref_logp`, and `weights`
    in fp32 or bool; they are constants and must not ask for a gradient.  With "mean" the weights add up to 2^-126 at
    least, or to zero: the gradient's divisor is fp32.  Columns from `vocab` on are padding.  Differentiable in
    the logits, which stay as they are (the gradient has memory of its own); once only."""
    if reduction not in ("mean", "sum"):
        raise ValueError(f"fused_policy_loss: reduction is 'mean' or 'sum' (got {reduction!r})")
    low, high = clip
    if logits.is_cuda:
        out = _ext.load().policy_loss(logits, tokens, old_logp, advantages, ref_logp, weights, low, high, kl_coef, vocab, reduction == "mean")
        if out is not None:
            return out
    # Not taken by the kernels: say why.
    if logits.dim() != 2 or logits.dtype not in _LOGITS or logits.shape[1] == 0 or logits.shape[0] >= 2 ** 31 or logits.shape[1] >= 2 ** 31 - 2 ** 16:
        raise ValueError(f"fused_policy_loss: logits are a bf16, fp16 or fp32 matrix (got {logits.dtype} {tuple(logits.shape)})")
    if not (low >= 0 and high >= 0):
        raise ValueError(f"fused_policy_loss: clip is two numbers from zero on (got {clip})")
    vocab = logits.shape[1] if vocab is None else vocab
    if not 0 < vocab <= logits.shape[1]:
        raise ValueError(f"fused_policy_loss: vocab {vocab} is outside 1 to {logits.shape[1]}")
    if kl_coef != 0 and ref_logp is None:
        raise ValueError("fused_policy_loss: kl_coef without ref_logp")
    rows = logits.shape[0]
    for name, t, kinds in (("tokens", tokens, (torch.int64,)), ("old_logp", old_logp, (torch.float32,)), ("advantages", advantages, (torch.float32,)),
                           ("ref_logp", ref_logp, (torch.float32,)), ("weights", weights, (torch.float32, torch.bool))):
        if t is None:
            continue
        if t.dtype not in kinds or t.shape != (rows,) or t.device != logits.device:
            raise ValueError(f"fused_policy_loss: {name} is {' or '.join(str(k) for k in kinds)} [{rows}] on {logits.device} "
                             f"(got {t.dtype} {list(t.shape)} on {t.device})")
        if t.requires_grad:
            raise ValueError(f"fused_policy_loss: {name} is a constant: detach it")
    if not logits.is_cuda:
        raise RuntimeError("fused_policy_loss runs on CUDA (sm_100a) only")
    raise RuntimeError("fused_policy_loss does not run under tracing, a dispatch mode or torch.func")
