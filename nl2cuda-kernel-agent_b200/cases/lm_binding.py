"""The torch binding of the language-model operators (csrc/binding/lm_torch.cpp over the C ABI of
include/lm_sm100.h), shared by layernorm, token_logprob, preference_loss, policy_loss and
orthogonalize.

It checks arguments (RuntimeError), takes outputs and workspaces from torch's caching allocator,
launches on torch's current stream of the operands' device, and holds the autograd nodes.  There is
no fallback: a missing library or a device that is not sm_100 raises.
"""
import functools

from framework.loader import load_torch_binding


@functools.cache
def ext():
    """The extension module (built on first use when a source is newer)."""
    return load_torch_binding()
