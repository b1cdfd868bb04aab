"""Token log-probabilities (``lp_sm100_*``, include/lm_sm100.h) for torch tensors, without autograd."""
from cases.lm_binding import ext


def logprob_forward(logits, labels, ignore_index, keep=True):
    """(logprob, stats): logprob (fp32) of labels' shape, 0 where the label is ``ignore_index``,
    and the [rows, 2] row statistics for ``logprob_backward`` (None unless ``keep``)."""
    return ext().logprob_forward(logits, labels, ignore_index, keep)


def logprob_backward(logits, labels, stats, coef, ignore_index):
    """dlogits = coef * (onehot(label) - softmax), with the stats of ``logprob_forward``; coef fp32
    of labels' shape."""
    return ext().logprob_backward(logits, labels, stats, coef, ignore_index)
