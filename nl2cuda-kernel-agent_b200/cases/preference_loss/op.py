"""The preference-loss candidate: autograd op over the sm_100a kernels.

``preference_loss(...)`` is the call for training programs; ``candidate(inputs, params)`` is the
harness contract.  The gradient flows to the logits.
"""
import torch
from torch.autograd.function import once_differentiable

from cases.preference_loss import native
from cases.token_logprob.native import logprob_backward


class PreferenceLossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ref_logprob, beta, label_smoothing, ignore_index):
        loss, reward, stats, coef = native.preference_forward(
            logits, labels, ref_logprob, beta, label_smoothing, ignore_index)
        ctx.save_for_backward(logits, labels, stats, coef)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(reward)
        return loss, reward

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _reward):
        logits, labels, stats, coef = ctx.saved_tensors
        dx = logprob_backward(logits, labels, stats, coef, ctx.ignore_index, scale0=g)
        return dx, None, None, None, None, None


def preference_loss(logits, labels, ref_logprob, beta=0.1, label_smoothing=0.0,
                    ignore_index=-100):
    """(loss, reward): the preference loss of B = 2P answers, answer p preferred to answer P + p,
    and each answer's reward [B] (not differentiable).

    logits [B, T, V] (CUDA; float32, bfloat16 or float16), labels [B, T] int64, ref_logprob
    [B, T] float32: the reference model's ``token_logprob`` of the same labels."""
    return PreferenceLossFunction.apply(logits, labels, ref_logprob, beta, label_smoothing,
                                        ignore_index)


def candidate(inputs, params):
    """Harness contract: inputs = {"logits", "labels", "ref_logprob"} -> loss."""
    return preference_loss(inputs["logits"], inputs["labels"], inputs["ref_logprob"],
                           params["beta"], params["label_smoothing"], params["ignore_index"])[0]


def forward_only(inputs, params):
    """Forward without autograd."""
    return native.preference_forward(inputs["logits"], inputs["labels"], inputs["ref_logprob"],
                                     params["beta"], params["label_smoothing"],
                                     params["ignore_index"])[0]
