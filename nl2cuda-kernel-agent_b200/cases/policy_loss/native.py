"""Clipped policy loss through the C ABI (``policy_sm100_loss``, include/lm_sm100.h) for torch
tensors."""
import torch

from cases import lm_binding as _lm
from cases.preference_loss.native import scores_like
from cases.token_logprob.native import logprob_forward


def policy_forward(logits, labels, old_logprob, ref_logprob, advantage, clip_low, clip_high,
                   kl_coef, ignore_index):
    """(loss [], kl [], stats, coef, norm): the loss, the mean KL estimate, the row statistics of
    the logits, and coef [B, T] and norm [], whose product is d loss / d logprob, for
    ``logprob_backward``."""
    if logits.dim() != 3:
        raise RuntimeError("logits must have shape [B, T, V]")
    lp, stats = logprob_forward(logits, labels, ignore_index)
    old = scores_like(old_logprob, labels, "old_logprob")
    ref = scores_like(ref_logprob, labels, "ref_logprob")
    per_token = advantage.dim() == 2
    _lm.check_cuda(("labels", "advantage"), (labels, advantage))
    if advantage.dtype != torch.float32 or advantage.shape != labels.shape[:advantage.dim()] \
            or advantage.dim() not in (1, 2):
        raise RuntimeError("advantage must be float32 with shape [B] or [B, T]")
    if advantage.requires_grad:
        raise RuntimeError("advantage is a constant of the loss: it must not require a gradient")
    adv = advantage.contiguous()
    labels = labels.contiguous()
    B, T = labels.shape
    dev = logits.device
    loss, kl, norm = (torch.empty((), dtype=torch.float32, device=dev) for _ in range(3))
    coef = torch.empty_like(lp)
    size = _lm.lib().loss_sm100_workspace_bytes(B, T)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _lm.call("policy_sm100_loss", dev, _lm.ptr(lp), _lm.ptr(old), _lm.ptr(ref), _lm.ptr(adv),
             int(per_token), _lm.ptr(labels), _lm.ptr(loss), _lm.ptr(kl), _lm.ptr(coef),
             _lm.ptr(norm), B, T, float(clip_low), float(clip_high), float(kl_coef),
             int(ignore_index), _lm.ptr(ws), size)
    return loss, kl, stats, coef, norm
