"""PyTorch definition of the token log-probability: the correctness standard of the Case, and the
base of the two losses' definitions.  The backward is torch autograd."""
import torch

from cases.token_logprob import config


def logprob(logits, labels, ignore_index):
    """log softmax(logits)[label] in at least fp32, 0 where the label is ``ignore_index``."""
    x = logits if logits.dtype == torch.float64 else logits.float()
    x = x - x.amax(dim=-1, keepdim=True).detach()
    scored = labels != ignore_index
    at = torch.where(scored, labels, 0).unsqueeze(-1)
    lp = x.gather(-1, at).squeeze(-1) - torch.log(torch.exp(x).sum(dim=-1))
    return torch.where(scored, lp, torch.zeros_like(lp))


def reference_forward(inputs, params):
    """inputs = {"logits" [B,T,V], "labels" [B,T]}, params = {"ignore_index"} -> [B,T]."""
    return logprob(inputs["logits"], inputs["labels"], params["ignore_index"])


def draw(gen, dtype, device, B, T, V, ignore_index):
    """Logits in which the label stands out, and labels with an unscored prompt and padding."""
    labels = torch.randint(0, V, (B, T), device=device, generator=gen)
    logits = 2.0 * torch.randn(B, T, V, device=device, generator=gen)
    boost = 6.0 + 2.0 * torch.randn(B, T, 1, device=device, generator=gen)
    logits.scatter_add_(2, labels.unsqueeze(-1), boost)
    u = torch.rand(2, B, 1, device=device, generator=gen)
    at = torch.arange(T, device=device).unsqueeze(0)
    inside = (at >= (u[0] * (T // 4 + 1)).floor()) & (at < T - (u[1] * (T // 4 + 1)).floor())
    return logits.to(dtype), torch.where(inside, labels, ignore_index)


def make_inputs(seed, dtype, device, requires_grad=False):
    """Named inputs {"logits", "labels"} for ``seed`` at the configured shape."""
    g = torch.Generator(device=device).manual_seed(seed)
    logits, labels = draw(g, dtype, device, config.B, config.T, config.V, config.IGNORE_INDEX)
    return {"logits": logits.requires_grad_(requires_grad), "labels": labels}
