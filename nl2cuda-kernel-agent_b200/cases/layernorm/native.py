"""Layer norm through the C ABI (``ln_sm100_*``, include/lm_sm100.h) for torch tensors."""
import math

import torch

from cases import lm_binding as _lm


def rows_of(t, D):
    """``t`` [..., D] as [rows, D] with contiguous rows: a view where its strides allow one."""
    t = t.reshape(math.prod(t.shape[:-1]), D)
    if (t.size(1) > 1 and t.stride(1) != 1) or (t.size(0) > 1 and t.stride(0) < D):
        t = t.contiguous()
    return t


def _check_parameters(x, weight, bias):
    if x.dim() == 0:
        raise RuntimeError("x must have at least one dimension")
    given = [(n, t) for n, t in (("weight", weight), ("bias", bias)) if t is not None]
    _lm.check_cuda(["x"] + [n for n, _ in given], [x] + [t for _, t in given])
    dtype = _lm.dtype_code(x, "x")
    for n, t in given:
        if tuple(t.shape) != (x.size(-1),):
            raise RuntimeError(f"{n} must have shape [{x.size(-1)}], not {list(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"{n} must have x's type or float32, not {t.dtype}")
    if len(given) == 2 and weight.dtype != bias.dtype:
        raise RuntimeError("weight and bias must have the same type")
    return dtype, _lm.DTYPES[given[0][1].dtype] if given else dtype


def ln_forward(x, weight, bias, eps, keep=True):
    """(y, mean, rstd) of x [..., D]; weight and bias [D] or None.  mean and rstd (fp32, one per
    row) are for ``ln_backward``; ``keep=False`` leaves them out (None)."""
    dtype, wdtype = _check_parameters(x, weight, bias)
    D = x.size(-1)
    rows = rows_of(x, D)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    n = rows.size(0)
    stats = torch.empty((2, n), dtype=torch.float32, device=x.device) if keep else None
    mean, rstd = (stats[0], stats[1]) if keep else (None, None)
    _lm.call("ln_sm100_forward", x.device, _lm.ptr(rows), rows.stride(0), _lm.ptr(weight),
             _lm.ptr(bias), _lm.ptr(y), _lm.ptr(mean), _lm.ptr(rstd), n, D, float(eps), dtype,
             wdtype)
    return y, mean, rstd


def ln_backward(dy, x, weight, mean, rstd, need=(True, True, True), wdtype=None):
    """[dx, dweight, dbias] (None where ``need`` is false) of sum(dy * y), with the mean and rstd
    of ``ln_forward``.  ``wdtype``: the type of dweight and dbias (default: weight's, or x's)."""
    D = x.size(-1)
    _lm.check_cuda(("dy", "x"), (dy, x))
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise RuntimeError("dy must have x's shape and type")
    dtype, _ = _check_parameters(x, weight, None)
    wdtype = wdtype or (weight.dtype if weight is not None else x.dtype)
    if weight is not None and weight.dtype != wdtype:
        raise RuntimeError("dweight and dbias have weight's type")
    rx, rdy = rows_of(x, D), rows_of(dy, D)
    n = rx.size(0)
    if mean.numel() != n or rstd.numel() != n:
        raise RuntimeError("mean and rstd must hold one value per row of x")
    weight = None if weight is None else weight.contiguous()
    dev = x.device
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need[0] else None
    dw = torch.empty(D, dtype=wdtype, device=dev) if need[1] else None
    db = torch.empty(D, dtype=wdtype, device=dev) if need[2] else None
    ws, size = None, 0
    if need[1] or need[2]:
        size = _lm.lib().ln_sm100_backward_workspace_bytes(n, D)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _lm.call("ln_sm100_backward", dev, _lm.ptr(rdy), rdy.stride(0), _lm.ptr(rx), rx.stride(0),
             _lm.ptr(weight), _lm.ptr(mean), _lm.ptr(rstd), _lm.ptr(dx), _lm.ptr(dw), _lm.ptr(db),
             n, D, dtype, _lm.DTYPES[wdtype], _lm.ptr(ws), size)
    return [dx, dw, db]
