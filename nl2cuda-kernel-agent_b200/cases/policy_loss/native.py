"""The clipped policy loss (``policy_sm100_loss``, include/lm_sm100.h) for torch tensors, without
autograd."""
from cases.lm_binding import ext


def policy_forward(logits, labels, old_logprob, ref_logprob, advantage, clip_low, clip_high,
                   kl_coef, ignore_index):
    """(loss [], kl [], state): state is what ``policy_backward`` needs."""
    return ext().policy_forward(logits, labels, old_logprob, ref_logprob, advantage, clip_low,
                                clip_high, kl_coef, ignore_index)


def policy_backward(logits, labels, state, g, ignore_index):
    """dlogits of g * loss (g: one fp32 on the device, or None for 1)."""
    return ext().loss_backward(logits, labels, state, g, True, ignore_index)
