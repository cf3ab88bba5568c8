"""Log probabilities of given labels, with each row's entropy and its most probable classes.

The loss beside the classification heads (model/decoder.py:120: log_softmax and argmax over
the classes): one pass over the logits gives what a training loss, a confidence and a list of
alternatives need, and the gradient recomputes the probabilities from the logits, so nothing of
the logits' size is kept between the two (pin_label_logprob, pin_label_logprob_bwd).  Both,
and the node in torch's graph, are called natively (csrc/pin_torch.cpp): small calls are the host's.
"""
from collections import namedtuple

import torch

from . import _lib

_NO_CLASS = (1 << 63) - 1
LabelLogProbs = namedtuple("LabelLogProbs", ["log_prob", "entropy", "top_log_prob", "top_index"])


def label_log_probs(logits: torch.Tensor, labels: torch.Tensor, top_k: int = 0, ignore_index: int = -100):
    """logits [..., C] (float32, float16 or bfloat16), labels [...] (whole numbers) ->
    LabelLogProbs(log_prob [...], entropy [...], top_log_prob [..., top_k], top_index [..., top_k]).

    log_prob, entropy (natural logarithms) and top_log_prob are float32 and differentiable with
    respect to the logits, once; top_index is int64, ties go to the lower class.  Rows whose label
    is ignore_index have log_prob 0 and pass no gradient through it.  Classes at -inf have
    probability 0; a row with nothing else has log_prob -inf, entropy 0 and gradient 0, a row with
    a NaN or +inf has NaN and top_index -1, a label outside [0, C) has log_prob NaN.  Rows may be
    strided (a slice of padded logits is read where it lies).  torch.func's transforms (vmap, grad,
    jvp, functionalize), forward-mode differentiation and fake tensors are refused; torch.compile
    breaks its graph here and calls this eagerly."""
    _lib.require_device(logits)
    if logits.dtype not in _lib.TYPES:
        raise ValueError(f"label_log_probs: logits must be float32, float16 or bfloat16 (got {logits.dtype})")
    if logits.dim() < 1 or labels.shape != logits.shape[:-1]:
        raise ValueError(f"label_log_probs: labels {tuple(labels.shape)} must have the logits' shape "
                         f"{tuple(logits.shape)} without its last dimension")
    if labels.device != logits.device:
        raise ValueError(f"label_log_probs: labels on {labels.device}, logits on {logits.device}")
    if labels.is_floating_point() or labels.is_complex() or labels.dtype == torch.bool:
        raise ValueError(f"label_log_probs: labels must be whole numbers (got {labels.dtype})")
    c = logits.shape[-1]
    if not 1 <= c <= _lib.LABEL_CLASSES_MAX:
        raise ValueError(f"label_log_probs: 1 to {_lib.LABEL_CLASSES_MAX} classes (got {c})")
    k = int(top_k)
    if not 0 <= k <= min(c, _lib.LABEL_TOP_MAX):
        raise ValueError(f"label_log_probs: top_k must be 0 to min(classes, {_lib.LABEL_TOP_MAX}) (got {top_k})")
    ignore = int(ignore_index)
    if not -(1 << 63) <= ignore < 1 << 63:
        raise ValueError(f"label_log_probs: ignore_index must fit in 64 bits with a sign (got {ignore_index})")
    z, y = logits, labels
    if logits.dim() != 2:
        z, y = logits.reshape(labels.numel(), c), labels.reshape(-1)
    if c > 1 and z.stride(1) != 1:
        z = z.contiguous()
    if z.is_neg():
        z = z.resolve_neg()
    if y.dtype == torch.uint64:   # beyond int64: no class, and not what ignore_index would be there
        y = y.to(torch.int64)
        y = torch.where(y < 0, _NO_CLASS - (ignore == _NO_CLASS), y)
    if y.dtype != torch.int64 or not y.is_contiguous() or y.is_neg():
        y = y.to(torch.int64).contiguous().resolve_neg()
    lp, ent, tlp, tidx = _lib.torch_fn("pin_torch_label")(
        _lib.address("pin_label_logprob_workspace_bytes"), _lib.address("pin_label_logprob"),
        _lib.address("pin_label_logprob_bwd"), z, y, k, ignore,
        1 if logits.requires_grad and torch.is_grad_enabled() else 0)
    if logits.dim() != 2:
        lead = labels.shape
        lp, ent, tlp, tidx = lp.view(lead), ent.view(lead), tlp.view(lead + (k,)), tidx.view(lead + (k,))
    return LabelLogProbs(lp, ent, tlp, tidx)
