"""ctypes binding of the language-model C ABI (include/lm_sm100.h), shared by the native modules
of layernorm, token_logprob, preference_loss, policy_loss and orthogonalize.

The library is the one of the RBF case (lib/librbf_sm100.so).  Kernels run on torch's current
stream of the operands' device; errors are raised as RuntimeError; there is no fallback: a
missing library or a non-sm_100 device raises.
"""
import ctypes
import threading

import torch

from cases.rbf import native as _rbf

_lock = threading.Lock()
_bound = None

_P = ctypes.c_void_p
_I = ctypes.c_int
_I64 = ctypes.c_int64
_F = ctypes.c_float
_SZ = ctypes.c_size_t

_SIGNATURES = {
    "ln_sm100_forward": (_I, [_P, _I64, _P, _P, _P, _P, _P, _I64, _I64, _F, _I, _I, _P]),
    "ln_sm100_backward_workspace_bytes": (_SZ, [_I64, _I64]),
    "ln_sm100_backward": (_I, [_P, _I64, _P, _I64, _P, _P, _P, _P, _P, _P, _I64, _I64, _I, _I,
                               _P, _SZ, _P]),
    "lp_sm100_forward": (_I, [_P, _I64, _I64, _P, _P, _P, _I64, _I64, _I64, _I64, _I, _P]),
    "lp_sm100_backward": (_I, [_P, _I64, _I64, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64,
                               _I, _P]),
    "loss_sm100_workspace_bytes": (_SZ, [_I64, _I64]),
    "pref_sm100_loss": (_I, [_P, _P, _P, _P, _P, _P, _I64, _I64, _F, _F, _I64, _P, _SZ, _P]),
    "policy_sm100_loss": (_I, [_P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _I64, _I64, _F, _F, _F,
                               _I64, _P, _SZ, _P]),
    "ortho_sm100_workspace_bytes": (_SZ, [_I64, _I64, _I64, _I]),
    "ortho_sm100": (_I, [_P, _I64, _I64, _P, _I64, _I64, _I64, ctypes.POINTER(_F), _I, _F, _I, _P,
                         _SZ, _P]),
}

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def lib():
    """The library with the signatures of include/lm_sm100.h declared."""
    global _bound
    if _bound is None:
        with _lock:
            if _bound is None:
                L = _rbf.lib()
                for name, (res, args) in _SIGNATURES.items():
                    fn = getattr(L, name)
                    fn.restype, fn.argtypes = res, args
                _bound = L
    return _bound


def dtype_code(t, name):
    """The ABI's element type of tensor ``t``."""
    code = DTYPES.get(t.dtype)
    if code is None:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    return code


def check_cuda(names, tensors):
    """Every tensor is on the GPU, and all on one."""
    for n, t in zip(names, tensors):
        if not t.is_cuda:
            raise RuntimeError(f"{n} must be a CUDA tensor")
        if t.device != tensors[0].device:
            raise RuntimeError(f"{', '.join(names)} must be on the same device")


def ptr(t):
    """The address of a tensor's data (None, or a tensor without elements: NULL)."""
    return t.data_ptr() if t is not None and t.numel() else None


def call(name, device, *args):
    """Call entry ``name`` with ``args`` and torch's current stream of ``device``, which is made
    the current device for the call; raise RuntimeError for a non-zero status."""
    fn = getattr(lib(), name)
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        status = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            status = fn(*args, stream)
    if status:
        _rbf.check(status, name)
