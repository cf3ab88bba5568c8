"""Log probabilities of given labels, with each row's entropy and its most probable classes.

The loss beside the classification heads (model/decoder.py:120: log_softmax and argmax over
the classes): one pass over the logits gives what a training loss, a confidence and a list of
alternatives need, and the gradient recomputes the probabilities from the logits, so nothing of
the logits' size is kept between the two (pin_label_logprob, pin_label_logprob_bwd).
"""
from collections import namedtuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib

LabelLogProbs = namedtuple("LabelLogProbs", ["log_prob", "entropy", "top_log_prob", "top_index"])


def _forward(z, y, k, ignore, want_stats):
    n, c = z.shape
    dev = z.device
    # one allocation for what is f32: the two columns, the statistics, the alternatives
    buf = torch.empty((2 * n * (1 + want_stats) + n * k,), dtype=torch.float32, device=dev)
    at = 2 * n * (1 + want_stats)
    lp, ent, stats, tlp = buf[:n], buf[n:2 * n], buf[2 * n:at] if want_stats else None, buf[at:].view(n, k)
    tidx = torch.empty((n, k), dtype=torch.int64, device=dev)
    dt = _lib.TYPES[z.dtype]
    base = buf.data_ptr()
    with _lib.on_device(dev):
        need = _lib.fn("pin_label_logprob_workspace_bytes")(n, c, dt, k)
        ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need > 0 else None
        _lib.call("pin_label_logprob", z.data_ptr(), dt, n, c, z.stride(0), y.data_ptr(), ignore, k, base, base + 4 * n,
                  base + 8 * n if want_stats else None, base + 4 * at if k else None, tidx.data_ptr() if k else None,
                  None if ws is None else ws.data_ptr(), _lib.stream(dev))
    return lp, ent, stats, tlp, tidx


class _LabelLogProbFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, y, k, ignore):
        ctx.set_materialize_grads(False)
        lp, ent, stats, tlp, tidx = _forward(z, y, k, ignore, True)
        ctx.save_for_backward(z, y, stats, ent, tidx)
        ctx.ignore = ignore
        ctx.mark_non_differentiable(tidx)
        return lp, ent, tlp, tidx

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, g_top, _):
        z, y, stats, ent, tidx = ctx.saved_tensors
        n, c = z.shape
        g_lp, g_ent, g_top = (None if g is None else g.to(torch.float32).contiguous() for g in (g_lp, g_ent, g_top))
        dz = torch.empty((n, c), dtype=z.dtype, device=z.device)
        with _lib.on_device(z.device):
            _lib.call("pin_label_logprob_bwd", z.data_ptr(), _lib.TYPES[z.dtype], n, c, z.stride(0), _lib.ptr(y),
                      ctx.ignore, tidx.shape[1], _lib.ptr(tidx), _lib.ptr(stats), _lib.ptr(ent), _lib.ptr(g_lp),
                      _lib.ptr(g_ent), _lib.ptr(g_top), _lib.ptr(dz), _lib.stream(z.device))
        return dz, None, None, None


def label_log_probs(logits: torch.Tensor, labels: torch.Tensor, top_k: int = 0, ignore_index: int = -100):
    """logits [..., C] (float32, float16 or bfloat16), labels [...] (whole numbers) ->
    LabelLogProbs(log_prob [...], entropy [...], top_log_prob [..., top_k], top_index [..., top_k]).

    log_prob, entropy (natural logarithms) and top_log_prob are float32 and differentiable with
    respect to the logits, once; top_index is int64, ties go to the lower class.  Rows whose label
    is ignore_index have log_prob 0 and pass no gradient through it.  Classes at -inf have
    probability 0; a row with nothing else has log_prob -inf, entropy 0 and gradient 0, a row with
    a NaN or +inf has NaN and top_index -1, a label outside [0, C) has log_prob NaN.  Rows may be
    strided (a slice of padded logits is read where it lies)."""
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
    lead = logits.shape[:-1]
    n = 1
    for s in lead:
        n *= s
    z = logits.reshape(n, c)
    if c > 1 and z.stride(1) != 1 or z.stride(0) < 0:
        z = z.contiguous()
    y = labels.reshape(n).to(torch.int64).contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        lp, ent, tlp, tidx = _LabelLogProbFn.apply(z, y, k, int(ignore_index))
    else:
        lp, ent, _, tlp, tidx = _forward(z.detach(), y, k, int(ignore_index), False)
    if len(lead) == 1:
        return LabelLogProbs(lp, ent, tlp, tidx)
    return LabelLogProbs(lp.view(lead), ent.view(lead), tlp.view(lead + (k,)), tidx.view(lead + (k,)))
