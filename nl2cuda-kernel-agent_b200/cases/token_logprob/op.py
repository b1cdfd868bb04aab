"""The token log-probability candidate: an autograd operator over the sm_100a kernels.

``token_logprob(logits, labels)`` is the call for models; ``candidate(inputs, params)`` is the
harness contract.  The gradient flows to the logits.
"""
from cases.lm_binding import ext
from cases.token_logprob import native


def token_logprob(logits, labels, ignore_index=-100):
    """log softmax(logits)[label] (float32, labels' shape), 0 where the label is ``ignore_index``.

    logits [..., V] (CUDA; float32, bfloat16 or float16), labels [...] int64.  A label outside
    [0, V) that is not ``ignore_index`` gives NaN."""
    return ext().token_logprob(logits, labels, ignore_index)


def candidate(inputs, params):
    """Harness contract: inputs = {"logits", "labels"}, params = {"ignore_index"} -> [B, T]."""
    return token_logprob(inputs["logits"], inputs["labels"], params["ignore_index"])


def forward_only(inputs, params):
    """Forward without autograd."""
    return native.logprob_forward(inputs["logits"], inputs["labels"], params["ignore_index"],
                                  keep=False)[0]
