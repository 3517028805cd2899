"""Training losses of the reference harness (src/run/kitti_seg.py:184-202, src/models/utils/lovasz_losses.py)
for device tensors, without the per-class host round trips of the reference loop.

The Lovasz-softmax term is evaluated for all classes at once: one segmented descending sort of the (C, P) error
matrix (device radix sort), two row-wise prefix sums, and a masked mean over the classes present -- no ``.sum() == 0``
sync per class (the reference does 20 of them on KITTI).
"""
from typing import NamedTuple, Optional

import torch
import torch.nn.functional as F

from ._lib import binding


def lovasz_softmax_flat(probas, labels, classes="present"):
    """ref lovasz_losses.py:174-202.  probas (P, C), labels (P,) in [0, C)."""
    if classes not in ("present", "all"):
        raise NotImplementedError("explicit class lists are not used by the reference harness")
    if probas.numel() == 0:
        return probas * 0.0
    p, c = probas.shape
    fg = F.one_hot(labels, c).to(probas.dtype).t().contiguous()            # (C, P) foreground masks
    err = (fg - probas.t()).abs()                                           # (C, P)
    err_sorted, order = torch.sort(err, dim=1, descending=True)
    fg_sorted = torch.gather(fg, 1, order)
    total = fg.sum(dim=1, keepdim=True)
    inter = total - fg_sorted.cumsum(1)
    union = total + (1.0 - fg_sorted).cumsum(1)
    jac = 1.0 - inter / union
    grad = torch.cat([jac[:, :1], jac[:, 1:] - jac[:, :-1]], dim=1)         # lovasz_grad (:19-31), constant w.r.t. probas
    per_class = (err_sorted * grad.detach()).sum(dim=1)
    if classes == "all":
        return per_class.mean()
    present = (total[:, 0] > 0).to(probas.dtype)
    return (per_class * present).sum() / present.sum()


class Scores(NamedTuple):
    """What token_logprobs returns; the last two are None where no alternatives were asked for."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: Optional[torch.Tensor]
    top_index: Optional[torch.Tensor]


def token_logprobs(logits, target, top=0, ignore_index=-100):
    """Log-probability of a given class in every row of ``logits`` (..., C), the row's entropy, and its ``top`` best alternatives,
    in one pass over the logits (ccn_logprob_fwd); differentiable with respect to the logits in logprob, entropy and top_logprob.

    logits: fp32, bf16 or fp16, any strides (columns that are not adjacent are copied).  target: int64 (or int32) of shape (...).
    top: 0 ... min(64, C).  Returns ``Scores``: logprob (...), entropy (...), top_logprob (..., top) in fp32 and top_index (...,
    top) in int64, best first, equal logits by ascending class.

    ``target == ignore_index``: logprob 0, no gradient from it; entropy and alternatives are the row's all the same.  Any other
    target outside [0, C): NaN, in logprob and (where logprob takes part in the loss) in the row's gradient.  Logits of -inf are
    classes without probability; a row of nothing else has logprob -inf, entropy 0 and gradient 0 but for the given class's own.
    The gradient has the logits' type, its rows 16-byte aligned (their stride padded where C is odd).  Where a backward pass is captured
    into a graph, no eager autograd graph of the same leaves may be alive, as for any torch operator."""
    return Scores(*binding().token_logprobs(logits, target, top, ignore_index))


def seg_loss_kitti(pred, gt, ignore=0, use_lovasz=False, class_weights=None):
    """ref kitti_seg.py:184-202: returns (loss, per-point NLL)."""
    logp = F.log_softmax(pred, dim=-1)
    if class_weights is None:
        per_point = F.nll_loss(logp, gt, reduction="none", ignore_index=ignore)
    else:
        assert ignore == 0
        w = torch.cat([torch.zeros(1, dtype=class_weights.dtype, device=class_weights.device), class_weights], dim=0)
        per_point = F.nll_loss(logp, gt, reduction="none", weight=w.to(pred.device))
    loss = per_point.mean()
    if use_lovasz:
        keep = gt != ignore
        loss = loss + 2 * lovasz_softmax_flat(F.softmax(pred, dim=-1)[keep], gt[keep]).mean()
    return loss, per_point
