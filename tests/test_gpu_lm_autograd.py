"""What the language-model operators do not differentiate is refused, never left out: gradients of
gradients, forward-mode tangents, and views that are negated lazily."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu

B, T, V, D = 2, 3, 40, 32


def operands():
    gen = torch.Generator(device="cuda").manual_seed(7)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    return {"x": randn(6, D), "weight": 1 + 0.1 * randn(D), "bias": 0.1 * randn(D),
            "logits": randn(B, T, V), "labels": torch.randint(0, V, (B, T), device="cuda", generator=gen),
            "old": -3 + 0.1 * randn(B, T), "ref": -3 + 0.1 * randn(B, T), "advantage": randn(B),
            "update": randn(8, 16)}


def calls():
    """name: (the call on a dict of operands, its tensors that carry numbers)."""
    from cases.layernorm.op import layer_norm
    from cases.orthogonalize.op import orthogonalize
    from cases.policy_loss.op import policy_loss
    from cases.preference_loss.op import preference_loss
    from cases.token_logprob.op import token_logprob
    return {
        "layer_norm": (lambda s: layer_norm(s["x"], s["weight"], s["bias"]), ("x", "weight", "bias")),
        "token_logprob": (lambda s: token_logprob(s["logits"], s["labels"]), ("logits",)),
        "preference_loss": (lambda s: preference_loss(s["logits"], s["labels"], s["ref"])[0], ("logits", "ref")),
        "policy_loss": (lambda s: policy_loss(s["logits"], s["labels"], s["old"], s["ref"], s["advantage"],
                                              kl_coef=0.1)[0], ("logits", "old", "ref", "advantage")),
        "orthogonalize": (lambda s: orthogonalize(s["update"]), ("update",)),
    }


DIFFERENTIABLE = [("layer_norm", "x"), ("token_logprob", "logits"), ("preference_loss", "logits"),
                  ("policy_loss", "logits")]


@pytest.mark.parametrize("name,leaf", DIFFERENTIABLE)
def test_gradient_of_a_gradient_penalty_is_refused(name, leaf, cuda_device):
    """A scalar's upstream gradient is a constant, but its gradient still depends on the operand: a penalty
    on it must not count as a constant."""
    call, s = calls()[name][0], operands()
    s[leaf].requires_grad_(True)
    loss = call(s).sum()
    (g,) = torch.autograd.grad(loss, s[leaf], create_graph=True)
    assert g.requires_grad
    with pytest.raises(RuntimeError, match="differentiated twice"):
        (loss + g.square().sum()).backward()


def test_gradient_of_parameters_gradients_is_refused(cuda_device):
    """dweight depends on x, and dx on weight; dbias on neither."""
    from cases.layernorm.op import layer_norm
    s = operands()
    for k in ("x", "weight", "bias"):
        s[k].requires_grad_(True)
    y = layer_norm(s["x"], s["weight"], s["bias"]).sum()
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), create_graph=True)
    assert dx.requires_grad and dw.requires_grad and not db.requires_grad
    for g in (dx, dw):
        with pytest.raises(RuntimeError, match="differentiated twice"):
            g.sum().backward(retain_graph=True)
    # With x a constant, dweight is one too; dx is not asked for.
    y = layer_norm(s["x"].detach(), s["weight"], s["bias"]).sum()
    dw, db = torch.autograd.grad(y, (s["weight"], s["bias"]), create_graph=True)
    assert not dw.requires_grad and not db.requires_grad
    # With weight alone of the two, dx still depends on x.
    y = layer_norm(s["x"], s["weight"].detach(), None).sum()
    (dx,) = torch.autograd.grad(y, s["x"], create_graph=True)
    assert dx.requires_grad


@pytest.mark.parametrize("name,leaf", DIFFERENTIABLE)
def test_first_gradients_stay_plain(name, leaf, cuda_device):
    """Without create_graph a gradient carries no graph, and it equals the one with it."""
    call, s = calls()[name][0], operands()
    s[leaf].requires_grad_(True)
    (g,) = torch.autograd.grad(call(s).sum(), s[leaf])
    assert not g.requires_grad
    (h,) = torch.autograd.grad(call(s).sum(), s[leaf], create_graph=True)
    assert torch.equal(g, h)
    call(s).sum().backward()
    assert torch.equal(s[leaf].grad, g) and not s[leaf].grad.requires_grad


@pytest.mark.parametrize("name", ["layer_norm", "token_logprob", "preference_loss", "policy_loss", "orthogonalize"])
def test_forward_mode_is_refused(name, cuda_device):
    call, names = calls()[name]
    for k in names:
        s = operands()
        with fwad.dual_level():
            s[k] = fwad.make_dual(s[k], torch.ones_like(s[k]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(s)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(s)
    s = operands()
    with fwad.dual_level():  # a level alone changes nothing
        got = call(s)
    assert torch.equal(got, call(s))


@pytest.mark.parametrize("name,leaf", [DIFFERENTIABLE[0], DIFFERENTIABLE[1]])
def test_tangent_of_an_upstream_gradient_is_refused(name, leaf, cuda_device):
    call, s = calls()[name][0], operands()
    s[leaf].requires_grad_(True)
    y = call(s)
    with fwad.dual_level():
        up = fwad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, s[leaf], up)


@pytest.mark.parametrize("name", ["layer_norm", "token_logprob", "preference_loss", "policy_loss", "orthogonalize"])
def test_lazily_negated_views(name, cuda_device):
    """The bytes of such a view have the other sign: refused; resolved, it is taken."""
    call, names = calls()[name]
    for k in names:
        s = operands()
        s[k] = torch._neg_view(s[k])
        with pytest.raises(RuntimeError, match="negated"):
            call(s)
        s[k] = s[k].resolve_neg()
        call(s)
