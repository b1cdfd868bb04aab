"""The preference loss (``pref_sm100_loss``, include/lm_sm100.h) for torch tensors, without
autograd."""
from cases.lm_binding import ext


def preference_forward(logits, labels, ref_logprob, beta, label_smoothing, ignore_index):
    """(loss [], reward [B], state): state is what ``preference_backward`` needs."""
    return ext().preference_forward(logits, labels, ref_logprob, beta, label_smoothing,
                                    ignore_index)


def preference_backward(logits, labels, state, g, ignore_index):
    """dlogits of g * loss (g: one fp32 on the device, or None for 1)."""
    return ext().loss_backward(logits, labels, state, g, False, ignore_index)
