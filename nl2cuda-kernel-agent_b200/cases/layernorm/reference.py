"""PyTorch definition of layer norm: the correctness standard of the Case.

``reference_forward`` takes the mean and the variance apart, in elementary operations and in at least
fp32, and rounds once; its backward is torch autograd.
"""
import torch

from cases.layernorm import config


def reference_forward(inputs, params):
    """inputs = {"x": [..., D], "weight": [D], "bias": [D]}, params = {"eps"} -> y."""
    dtype = inputs["x"].dtype
    x, weight, bias = (t if t.dtype == torch.float64 else t.float()
                       for t in (inputs["x"], inputs["weight"], inputs["bias"]))
    c = x - x.mean(dim=-1, keepdim=True)
    var = c.pow(2).mean(dim=-1, keepdim=True)
    return (c / torch.sqrt(var + params["eps"]) * weight + bias).to(dtype)


def make_inputs(seed, dtype, device, requires_grad=False):
    """Named inputs {"x", "weight", "bias"} for ``seed`` at the configured shape."""
    g = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, dtype=torch.float32, device=device, generator=g)

    out = {"x": randn(config.ROWS, config.D).to(dtype),
           "weight": (1 + 0.1 * randn(config.D)).to(dtype),
           "bias": (0.1 * randn(config.D)).to(dtype)}
    if requires_grad:
        for t in out.values():
            t.requires_grad_(True)
    return out
