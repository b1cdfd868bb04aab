"""The layer-norm candidate: an autograd operator over the sm_100a kernels.

``layer_norm(x, weight, bias, eps)`` is the call for models; ``candidate(inputs, params)`` is the
harness contract.  Gradients flow to x, weight and bias.
"""
from cases.layernorm import native
from cases.lm_binding import ext


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x (CUDA tensor, float32,
    bfloat16 or float16); weight and bias [D], of x's type or float32, or None (1 and 0)."""
    return ext().layer_norm(x, weight, bias, eps)


def candidate(inputs, params):
    """Harness contract: inputs = {"x", "weight", "bias"}, params = {"eps"} -> y."""
    return layer_norm(inputs["x"], inputs["weight"], inputs["bias"], params["eps"])


def forward_only(inputs, params):
    """Forward without autograd."""
    return native.ln_forward(inputs["x"], inputs["weight"], inputs["bias"], params["eps"],
                             keep=False)[0]
