"""The preference-loss candidate: an autograd operator over the sm_100a kernels.

``preference_loss(...)`` is the call for training programs; ``candidate(inputs, params)`` is the
harness contract.  The gradient flows to the logits.
"""
from cases.lm_binding import ext
from cases.preference_loss import native


def preference_loss(logits, labels, ref_logprob, beta=0.1, label_smoothing=0.0,
                    ignore_index=-100):
    """(loss, reward): the preference loss of B = 2P answers, answer p preferred to answer P + p,
    and each answer's reward [B] (not differentiable).

    logits [B, T, V] (CUDA; float32, bfloat16 or float16), labels [B, T] int64, ref_logprob
    [B, T] float32: the reference model's ``token_logprob`` of the same labels."""
    return ext().preference_loss(logits, labels, ref_logprob, beta, label_smoothing, ignore_index)


def candidate(inputs, params):
    """Harness contract: inputs = {"logits", "labels", "ref_logprob"} -> loss."""
    return preference_loss(inputs["logits"], inputs["labels"], inputs["ref_logprob"],
                           params["beta"], params["label_smoothing"], params["ignore_index"])[0]


def forward_only(inputs, params):
    """Forward without autograd."""
    return native.preference_forward(inputs["logits"], inputs["labels"], inputs["ref_logprob"],
                                     params["beta"], params["label_smoothing"],
                                     params["ignore_index"])[0]
