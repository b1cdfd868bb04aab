"""Orthogonalisation (``ortho_sm100``, include/lm_sm100.h) for torch tensors."""
from cases.lm_binding import ext
from cases.orthogonalize.reference import per_step


def orthogonalize(update, steps, coefficients, eps):
    """The orthogonalised ``update`` [..., m, n] (CUDA; float32, bfloat16 or float16).  With
    RBF_CHECK_STATUS=1 the device status word is read after it (one synchronisation; not inside a
    capture), and a bounded device wait that ran out raises."""
    flat = [v for s in per_step(coefficients, int(steps)) for v in s]
    return ext().orthogonalize(update, flat, eps)
