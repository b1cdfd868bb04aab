"""Preference loss through the C ABI (``pref_sm100_loss``, include/lm_sm100.h) for torch tensors."""
import torch

from cases import lm_binding as _lm
from cases.token_logprob.native import logprob_forward


def scores_like(t, labels, name):
    """``t``, float32 of labels' shape on its device, contiguous."""
    _lm.check_cuda(("labels", name), (labels, t))
    if t.dtype != torch.float32 or t.shape != labels.shape:
        raise RuntimeError(f"{name} must be float32 with labels' shape {list(labels.shape)}")
    if t.requires_grad:
        raise RuntimeError(f"{name} is a constant of the loss: it must not require a gradient")
    return t.contiguous()


def preference_forward(logits, labels, ref_logprob, beta, label_smoothing, ignore_index):
    """(loss [], reward [B], stats, coef): the loss, the rewards, the row statistics of the
    logits and d loss / d logprob [B, T] for ``logprob_backward``."""
    if logits.dim() != 3:
        raise RuntimeError("logits must have shape [B, T, V]")
    if logits.size(0) % 2:
        raise RuntimeError("logits must hold pairs: B is odd")
    lp, stats = logprob_forward(logits, labels, ignore_index)
    ref = scores_like(ref_logprob, labels, "ref_logprob")
    labels = labels.contiguous()
    B, T = labels.shape
    dev = logits.device
    loss = torch.empty((), dtype=torch.float32, device=dev)
    reward = torch.empty(B, dtype=torch.float32, device=dev)
    coef = torch.empty_like(lp)
    size = _lm.lib().loss_sm100_workspace_bytes(B, T)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _lm.call("pref_sm100_loss", dev, _lm.ptr(lp), _lm.ptr(ref), _lm.ptr(labels), _lm.ptr(loss),
             _lm.ptr(reward), _lm.ptr(coef), B, T, float(beta), float(label_smoothing),
             int(ignore_index), _lm.ptr(ws), size)
    return loss, reward, stats, coef
