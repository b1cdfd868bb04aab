"""Layer norm's passes (``ln_sm100_*``, include/lm_sm100.h) for torch tensors, without autograd."""
from cases.lm_binding import ext


def ln_forward(x, weight, bias, eps, keep=True):
    """(y, stats) of x [..., D]; weight and bias [D] or None.  stats [2, rows] (fp32: the means and
    the reciprocal deviations) are for ``ln_backward``; ``keep=False`` leaves them out (None)."""
    return ext().ln_forward(x, weight, bias, float(eps), keep)


def ln_backward(dy, x, weight, stats, need=(True, True, True), like=None):
    """[dx, dweight, dbias] (None where ``need`` is false) of sum(dy * y), with the stats of
    ``ln_forward``.  dweight and dbias have weight's type, or without one that of ``like`` or x."""
    return ext().ln_backward(dy, x, weight, stats, need, like)
