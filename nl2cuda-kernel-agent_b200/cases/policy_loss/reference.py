"""PyTorch definition of the clipped policy loss: the correctness standard of the Case.  The
backward is torch autograd."""
import torch

from cases.policy_loss import config
from cases.token_logprob.reference import draw, logprob


def policy(lp, old_logprob, ref_logprob, advantage, labels, clip_low, clip_high, kl_coef,
           ignore_index):
    """(loss, kl) of log-probabilities [B, T], in fp64."""
    scored = labels != ignore_index
    count = scored.sum().clamp(min=1)
    a = advantage.double()
    a = a.unsqueeze(1) if a.dim() == 1 else a
    ratio = torch.exp(torch.where(scored, lp.double() - old_logprob.double(), 0.0))
    d = torch.where(scored, ref_logprob.double() - lp.double(), 0.0)
    kl = torch.exp(d) - d - 1
    gain = torch.minimum(ratio * a, ratio.clamp(1 - clip_low, 1 + clip_high) * a)
    terms = torch.where(scored, kl_coef * kl - gain, 0.0)
    return terms.sum() / count, kl.sum() / count


def reference_forward(inputs, params):
    """inputs = {"logits", "labels", "old_logprob", "ref_logprob", "advantage"}, params as
    ``CASE.params`` -> loss [] fp32."""
    lp = logprob(inputs["logits"], inputs["labels"], params["ignore_index"])
    loss, _ = policy(lp, inputs["old_logprob"], inputs["ref_logprob"], inputs["advantage"],
                     inputs["labels"], params["clip_low"], params["clip_high"],
                     params["kl_coef"], params["ignore_index"])
    return loss.float()


def make_inputs(seed, dtype, device, requires_grad=False):
    """Named inputs for ``seed`` at the configured shape."""
    g = torch.Generator(device=device).manual_seed(seed)
    logits, labels = draw(g, dtype, device, config.B, config.T, config.V, config.IGNORE_INDEX)
    lp = logprob(logits, labels, config.IGNORE_INDEX)
    scored = labels != config.IGNORE_INDEX

    def near(spread):
        return torch.where(scored, lp + spread * torch.randn(lp.shape, device=device,
                                                             generator=g), 0.0)

    return {"old_logprob": near(0.15), "ref_logprob": near(0.2),
            "advantage": torch.randn(config.B, device=device, generator=g), "labels": labels,
            "logits": logits.requires_grad_(requires_grad)}
