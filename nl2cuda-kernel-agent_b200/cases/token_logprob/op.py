"""The token log-probability candidate: autograd op over the sm_100a kernels.

``token_logprob(logits, labels)`` is the call for models; ``candidate(inputs, params)`` is the
harness contract.  The gradient flows to the logits.
"""
import torch
from torch.autograd.function import once_differentiable

from cases.token_logprob import native


class TokenLogprobFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ignore_index):
        lp, stats = native.logprob_forward(logits, labels, ignore_index)
        ctx.save_for_backward(logits, labels, stats)
        ctx.ignore_index = ignore_index
        return lp

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, labels, stats = ctx.saved_tensors
        return native.logprob_backward(logits, labels, stats, g, ctx.ignore_index), None, None


def token_logprob(logits, labels, ignore_index=-100):
    """log softmax(logits)[label] (float32, labels' shape), 0 where the label is ``ignore_index``.

    logits [..., V] (CUDA; float32, bfloat16 or float16), labels [...] int64.  A label outside
    [0, V) that is not ``ignore_index`` gives NaN."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobFunction.apply(logits, labels, ignore_index)
    return native.logprob_forward(logits, labels, ignore_index, keep=False)[0]


def candidate(inputs, params):
    """Harness contract: inputs = {"logits", "labels"}, params = {"ignore_index"} -> [B, T]."""
    return token_logprob(inputs["logits"], inputs["labels"], params["ignore_index"])


def forward_only(inputs, params):
    """Forward without autograd."""
    return native.logprob_forward(inputs["logits"], inputs["labels"], params["ignore_index"],
                                  keep=False)[0]
