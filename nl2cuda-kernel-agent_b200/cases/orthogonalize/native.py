"""Orthogonalisation through the C ABI (``ortho_sm100``, include/lm_sm100.h) for torch tensors."""
import ctypes

import torch

from cases import lm_binding as _lm
from cases.orthogonalize.reference import per_step
from cases.rbf.native import read_status
from cases.rbf.shard import check_status_default


def orthogonalize(update, steps, coefficients, eps):
    """The orthogonalised ``update`` [..., m, n] (CUDA; float32, bfloat16 or float16)."""
    _lm.check_cuda(("update",), (update,))
    dtype = _lm.dtype_code(update, "update")
    if update.dim() < 2:
        raise RuntimeError("update must have at least two dimensions")
    steps = int(steps)
    coef = per_step(coefficients, steps)
    m, n = update.shape[-2:]
    out = torch.empty(update.shape, dtype=update.dtype, device=update.device)
    if out.numel() == 0:
        return out
    g = update.reshape(-1, m, n)
    if (n > 1 and g.stride(2) != 1) or (m > 1 and g.stride(1) < n) or g.stride(0) < 0:
        g = g.contiguous()
    batch = g.size(0)
    size = _lm.lib().ortho_sm100_workspace_bytes(batch, m, n, steps)
    ws = torch.empty(size, dtype=torch.uint8, device=update.device)
    flat = (ctypes.c_float * (3 * steps))(*[v for s in coef for v in s])
    _lm.call("ortho_sm100", update.device, _lm.ptr(g), g.stride(1), g.stride(0), _lm.ptr(out), batch,
             m, n, flat, steps, float(eps), dtype, _lm.ptr(ws), size)
    if check_status_default():
        status = read_status(ws)
        if status != 0:
            raise RuntimeError(f"orthogonalize: device status {status} (a bounded device-side wait "
                               "timed out)")
    return out
