"""The clipped policy-loss candidate: an autograd operator over the sm_100a kernels.

``policy_loss(...)`` is the call for training programs; ``candidate(inputs, params)`` is the
harness contract.  The gradient flows to the logits.
"""
from cases.lm_binding import ext
from cases.policy_loss import native


def policy_loss(logits, labels, old_logprob, ref_logprob, advantage, clip_low=0.2, clip_high=0.2,
                kl_coef=0.0, ignore_index=-100):
    """(loss, kl): the clipped policy loss, a mean over all scored positions, and the mean KL
    estimate (not differentiable).

    logits [B, T, V] (CUDA; float32, bfloat16 or float16), labels [B, T] int64, old_logprob and
    ref_logprob [B, T] float32, advantage [B] or [B, T] float32."""
    return ext().policy_loss(logits, labels, old_logprob, ref_logprob, advantage, clip_low,
                             clip_high, kl_coef, ignore_index)


def candidate(inputs, params):
    """Harness contract: inputs = {"logits", "labels", "old_logprob", "ref_logprob",
    "advantage"} -> loss."""
    return policy_loss(inputs["logits"], inputs["labels"], inputs["old_logprob"],
                       inputs["ref_logprob"], inputs["advantage"], params["clip_low"],
                       params["clip_high"], params["kl_coef"], params["ignore_index"])[0]


def forward_only(inputs, params):
    """Forward without autograd."""
    return native.policy_forward(inputs["logits"], inputs["labels"], inputs["old_logprob"],
                                 inputs["ref_logprob"], inputs["advantage"],
                                 params["clip_low"], params["clip_high"], params["kl_coef"],
                                 params["ignore_index"])[0]
