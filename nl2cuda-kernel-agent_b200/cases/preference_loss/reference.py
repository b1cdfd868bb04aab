"""PyTorch definition of the preference loss: the correctness standard of the Case.  The backward
is torch autograd."""
import torch

from cases.preference_loss import config
from cases.token_logprob.reference import draw, logprob


def preference(lp, ref_logprob, labels, beta, label_smoothing, ignore_index):
    """(loss, reward) of log-probabilities [B, T]; sums over positions in fp64."""
    d = torch.where(labels != ignore_index, lp.double() - ref_logprob.double(), 0.0)
    reward = beta * d.sum(dim=1)
    P = reward.numel() // 2
    z = reward[:P] - reward[P:]
    log_sigmoid = torch.nn.functional.logsigmoid
    loss = -(1 - label_smoothing) * log_sigmoid(z) - label_smoothing * log_sigmoid(-z)
    return loss.mean(), reward


def reference_forward(inputs, params):
    """inputs = {"logits", "labels", "ref_logprob"}, params as ``CASE.params`` -> loss [] fp32."""
    lp = logprob(inputs["logits"], inputs["labels"], params["ignore_index"])
    loss, _ = preference(lp, inputs["ref_logprob"], inputs["labels"], params["beta"],
                         params["label_smoothing"], params["ignore_index"])
    return loss.float()


def make_inputs(seed, dtype, device, requires_grad=False):
    """Named inputs {"logits", "labels", "ref_logprob"} for ``seed`` at the configured shape."""
    g = torch.Generator(device=device).manual_seed(seed)
    logits, labels = draw(g, dtype, device, config.B, config.T, config.V, config.IGNORE_INDEX)
    lp = logprob(logits, labels, config.IGNORE_INDEX)
    ref = lp + 0.1 * torch.randn(lp.shape, device=device, generator=g)
    ref = torch.where(labels != config.IGNORE_INDEX, ref, 0.0)
    return {"logits": logits.requires_grad_(requires_grad), "labels": labels, "ref_logprob": ref}
