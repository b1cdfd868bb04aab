"""Token log-probabilities through the C ABI (``lp_sm100_*``, include/lm_sm100.h) for torch
tensors: the passes over the logits that token_logprob and both losses share."""
import torch

from cases import lm_binding as _lm


def check_logits(logits, labels):
    """The element type's code; raises for what the kernels do not take."""
    _lm.check_cuda(("logits", "labels"), (logits, labels))
    dtype = _lm.dtype_code(logits, "logits")
    if logits.dim() < 2:
        raise RuntimeError("logits must have shape [..., V] with at least one leading dimension")
    if labels.dtype != torch.int64:
        raise RuntimeError(f"labels must be int64, not {labels.dtype}")
    if labels.shape != logits.shape[:-1]:
        raise RuntimeError(f"labels must have shape {list(logits.shape[:-1])}, "
                           f"not {list(labels.shape)}")
    return dtype


def rows_of(logits):
    """(logits, batch stride, row stride, T): rows r at (r // T) * batch stride + (r % T) * row
    stride, for logits [B, T, V] of any strides with contiguous rows; anything else is copied."""
    V = logits.size(-1)
    if logits.dim() == 2:
        logits = logits.unsqueeze(0)
    if logits.dim() != 3:
        logits = logits.reshape(-1, logits.size(-2), V)
    if (V > 1 and logits.stride(2) != 1) or min(logits.stride()) < 0:
        logits = logits.contiguous()
    return logits, logits.stride(0), logits.stride(1), logits.size(1)


def logprob_forward(logits, labels, ignore_index, keep=True):
    """(logprob, stats): logprob (fp32) of labels' shape, 0 where the label is ``ignore_index``,
    and the [rows, 2] row statistics for ``logprob_backward`` (None unless ``keep``)."""
    dtype = check_logits(logits, labels)
    x, sb, st, T = rows_of(logits)
    labels = labels.contiguous()
    n, V, dev = labels.numel(), logits.size(-1), logits.device
    lp = torch.empty(labels.shape, dtype=torch.float32, device=dev)
    stats = torch.empty((n, 2), dtype=torch.float32, device=dev) if keep else None
    _lm.call("lp_sm100_forward", dev, _lm.ptr(x), sb, st, _lm.ptr(labels), _lm.ptr(lp),
             _lm.ptr(stats), n, T, V, int(ignore_index), dtype)
    return lp, stats


def logprob_backward(logits, labels, stats, coef, ignore_index, scale0=None, scale1=None):
    """dlogits = coef * scale0 * scale1 * (onehot(label) - softmax), with the stats of
    ``logprob_forward``; coef fp32 of labels' shape, the scales fp32 device scalars or None."""
    dtype = check_logits(logits, labels)
    x, sb, st, T = rows_of(logits)
    labels, coef = labels.contiguous(), coef.contiguous()
    n, V, dev = labels.numel(), logits.size(-1), logits.device
    if coef.dtype != torch.float32 or coef.numel() != n or stats.numel() != 2 * n:
        raise RuntimeError("coef and stats must be float32, one and two values per row")
    dx = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    _lm.call("lp_sm100_backward", dev, _lm.ptr(x), sb, st, _lm.ptr(labels), _lm.ptr(stats),
             _lm.ptr(coef), _lm.ptr(scale0), _lm.ptr(scale1), _lm.ptr(dx), n, T, V,
             int(ignore_index), dtype)
    return dx
