"""The C ABI of include/lm_sm100.h through ctypes, as a caller without torch binds it."""
import ctypes

_P = ctypes.c_void_p
_I = ctypes.c_int
_I64 = ctypes.c_int64
_F = ctypes.c_float
_SZ = ctypes.c_size_t

SIGNATURES = {
    "ln_sm100_forward": (_I, [_P, _I64, _P, _P, _P, _P, _P, _I64, _I64, _F, _I, _I, _P]),
    "ln_sm100_backward_workspace_bytes": (_SZ, [_I64, _I64]),
    "ln_sm100_backward": (_I, [_P, _I64, _P, _I64, _P, _P, _P, _P, _P, _P, _I64, _I64, _I, _I,
                               _P, _SZ, _P]),
    "lp_sm100_forward": (_I, [_P, _I64, _I64, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I, _P]),
    "lp_sm100_backward": (_I, [_P, _I64, _I64, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64,
                               _I, _P]),
    "loss_sm100_workspace_bytes": (_SZ, [_I64, _I64]),
    "pref_sm100_loss": (_I, [_P, _P, _P, _P, _P, _P, _P, _I64, _I64, _F, _F, _I64, _P, _SZ, _P]),
    "policy_sm100_loss": (_I, [_P, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _I64, _I64, _F, _F, _F,
                               _I64, _P, _SZ, _P]),
    "ortho_sm100_workspace_bytes": (_SZ, [_I64, _I64, _I64, _I]),
    "ortho_sm100": (_I, [_P, _I64, _I64, _P, _I64, _I64, _I64, ctypes.POINTER(_F), _I, _F, _I, _P,
                         _SZ, _P]),
}


def lib():
    from cases.rbf import native
    L = native.lib()
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(L, name)
        fn.restype, fn.argtypes = res, args
    return L
