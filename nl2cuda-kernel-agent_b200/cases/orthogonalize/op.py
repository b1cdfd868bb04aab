"""The orthogonalisation candidate over the sm_100a kernels.

``orthogonalize(update, ...)`` is the call for optimisers; ``candidate(inputs, params)`` is the
harness contract.  There is no gradient: an update is not differentiated.
"""
from cases.orthogonalize import config, native


def orthogonalize(update, steps=config.STEPS, coefficients=config.COEFFICIENTS, eps=config.EPS):
    """``update`` [..., m, n] with all its singular values brought near 1 by ``steps``
    Newton-Schulz products; coefficients (a, b, c), or one of these for every step.  Same shape and
    type (float32, bfloat16 or float16, CUDA); leading dimensions are a batch.  An update that
    requires a gradient is refused outside torch.no_grad()."""
    return native.orthogonalize(update, steps, coefficients, eps)


def candidate(inputs, params):
    """Harness contract: inputs = {"update"}, params = {"steps", "coefficients", "eps"}."""
    return orthogonalize(inputs["update"], params["steps"], params["coefficients"], params["eps"])


def forward_only(inputs, params):
    """Same: there is no autograd in this case."""
    return candidate(inputs, params)
