"""PyTorch definition of the orthogonalised update: the correctness standard of the Case."""
import torch

from cases.orthogonalize import config


def per_step(coefficients, steps):
    """One (a, b, c) for every step, from one for all of them or a list of ``steps``."""
    c = list(coefficients)
    if len(c) == 3 and not any(hasattr(v, "__len__") for v in c):
        c = [c] * steps
    if len(c) != steps or any(len(v) != 3 for v in c):
        raise RuntimeError("coefficients must be (a, b, c), or one of these for every step")
    return [tuple(float(v) for v in s) for s in c]


def reference_forward(inputs, params):
    """inputs = {"update" [..., m, n]}, params as ``CASE.params`` -> the orthogonalised update."""
    x = inputs["update"]
    dtype = x.dtype
    if dtype != torch.float64:
        x = x.float()
    tall = x.size(-2) > x.size(-1)
    if tall:
        x = x.mT
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + params["eps"])
    for a, b, c in per_step(params["coefficients"], params["steps"]):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return (x.mT if tall else x).to(dtype)


def make_inputs(seed, dtype, device, requires_grad=False):
    """Named inputs {"update"} for ``seed`` at the configured shape: some strong directions that
    fall off, and noise.  (An update takes no gradient; ``requires_grad`` is ignored.)"""
    g = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=device, generator=g)

    k = min(config.M, config.N, 16)
    fall = 1.0 / torch.arange(1, k + 1, device=device)
    u = (randn(config.M, k) * fall) @ randn(k, config.N) + 0.5 * randn(config.M, config.N)
    return {"update": (1e-3 * u).to(dtype)}
