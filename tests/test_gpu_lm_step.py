"""The language-model operators together, as a fine-tuning step uses them: hidden states through a
layer norm and a projection to logits, a preference or a policy loss on them, the backward pass, and
the projection moved by its orthogonalised gradient.  Against the same step in 64 bits."""
import math

import pytest
import torch

from lm_util import U32

pytestmark = pytest.mark.gpu

IGNORE = -100


def inputs(B, T, D, V, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=g)

    labels = torch.randint(0, V, (B, T), device="cuda", generator=g)
    labels[:, :2] = IGNORE
    labels[1, -3:] = IGNORE
    return {"hidden": randn(B, T, D), "weight": 1 + 0.1 * randn(D), "bias": 0.1 * randn(D),
            "head": randn(V, D) / math.sqrt(D), "ref_head": randn(V, D) / math.sqrt(D),
            "labels": labels, "advantage": randn(B)}


def step(s, which, ops):
    """One step with the operators in ``ops``: (loss, extra, gradients, new head)."""
    leaves = {k: s[k].clone().requires_grad_(True) for k in ("hidden", "weight", "bias", "head")}
    h = ops["norm"](leaves["hidden"], leaves["weight"], leaves["bias"])
    logits = h @ leaves["head"].T
    with torch.no_grad():
        ref = ops["logprob"](h @ s["ref_head"].T.to(h.dtype), s["labels"])
        old = ops["logprob"](logits * 0.9, s["labels"])
    if which == "preference":
        loss, extra = ops["preference"](logits, s["labels"], ref)
    else:
        loss, extra = ops["policy"](logits, s["labels"], old, ref, s["advantage"])
    loss.backward()
    with torch.no_grad():
        head = leaves["head"] - 0.1 * ops["orthogonalize"](leaves["head"].grad)
    return loss.detach(), extra.detach(), {k: v.grad for k, v in leaves.items()}, head


def own_ops():
    from cases.layernorm.op import layer_norm
    from cases.orthogonalize.op import orthogonalize
    from cases.policy_loss.op import policy_loss
    from cases.preference_loss.op import preference_loss
    from cases.token_logprob.op import token_logprob
    return {"norm": lambda x, w, b: layer_norm(x, w, b, 1e-5), "logprob": token_logprob,
            "preference": lambda x, lab, ref: preference_loss(x, lab, ref, 0.1, 0.05),
            "policy": lambda x, lab, old, ref, a: policy_loss(x, lab, old, ref, a, 0.2, 0.2, 0.1),
            "orthogonalize": orthogonalize}


def plain_ops():
    from cases.orthogonalize.reference import reference_forward as ortho
    from cases.policy_loss.reference import policy
    from cases.preference_loss.reference import preference
    from cases.token_logprob.reference import logprob

    def preference_of(x, lab, ref):
        return preference(logprob(x, lab, IGNORE), ref, lab, 0.1, 0.05, IGNORE)

    def policy_of(x, lab, old, ref, a):
        return policy(logprob(x, lab, IGNORE), old, ref, a, lab, 0.2, 0.2, 0.1, IGNORE)

    params = {"steps": 5, "coefficients": (3.4445, -4.7750, 2.0315), "eps": 1e-7}
    return {"norm": lambda x, w, b: torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, 1e-5),
            "logprob": lambda x, lab: logprob(x, lab, IGNORE), "preference": preference_of,
            "policy": policy_of, "orthogonalize": lambda g: ortho({"update": g}, params)}


@pytest.mark.parametrize("which", ["preference", "policy"])
def test_step_against_64_bits(which, cuda_device):
    s = inputs(4, 24, 96, 1500, 3)
    got = step(s, which, own_ops())
    want = step({k: v.double() if v.is_floating_point() else v for k, v in s.items()}, which,
                plain_ops())
    # fp32 throughout: the projections' sums of 96 and 1500 products and the operators' own errors
    # are each within some 100 roundings of their largest terms, about 10 times the results here.
    tol = 1000 * U32
    assert abs(float(got[0]) - float(want[0])) <= tol * (1 + abs(float(want[0])))
    assert float((got[1].double() - want[1]).abs().max()) <= tol * (1 + float(want[1].abs().max()))
    for k in got[2]:
        scale = float(want[2][k].abs().max())
        assert float((got[2][k].double() - want[2][k]).abs().max()) <= tol * scale, k
    # The orthogonalised gradient multiplies its errors with the small singular values, by up to
    # 3.4445^5 = 485: within that of the gradient's own relative error, and far above it by chance only.
    moved = want[3] - s["head"].double()
    off = (got[3] - s["head"]).double() - moved
    assert float(off.norm()) <= 485 * tol * float(moved.norm())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_step_in_16_bits_runs_and_moves_the_head(dtype, cuda_device):
    s = {k: v.to(dtype) if v.is_floating_point() and k != "advantage" else v
         for k, v in inputs(2, 40, 256, 1031, 4).items()}
    loss, extra, grads, head = step(s, "policy", own_ops())
    assert torch.isfinite(loss) and torch.isfinite(extra).all()
    assert all(torch.isfinite(g).all() and g.any() for g in grads.values())
    assert head.dtype == dtype and torch.isfinite(head).all()
    sv = torch.linalg.svdvals(((s["head"] - head).double() / 0.1))
    assert float(sv.max()) < 1.4


def test_gradients_of_broadcast_and_shared_operands(cuda_device):
    """One weight used by two norms, and one row of hidden states expanded to many."""
    from cases.layernorm.op import layer_norm
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1, 64, device="cuda", generator=g, requires_grad=True)
    w = torch.randn(64, device="cuda", generator=g, requires_grad=True)
    a = layer_norm(x.expand(50, 64), w, None, 1e-5)
    b = layer_norm(a, w, None, 1e-5)
    up = torch.randn(50, 64, device="cuda", generator=g)
    (b * up).sum().backward()
    x64, w64 = (t.detach().double().requires_grad_(True) for t in (x, w))
    f = torch.nn.functional.layer_norm
    a = f(x64.expand(50, 64), (64,), w64, None, 1e-5)
    (f(a, (64,), w64, None, 1e-5) * up.double()).sum().backward()
    for t, r in ((x.grad, x64.grad), (w.grad, w64.grad)):
        assert float((t.double() - r).abs().max()) <= 2000 * U32 * float(r.abs().max())


def test_second_derivative_is_refused(cuda_device):
    from cases.layernorm.op import layer_norm
    from cases.token_logprob.op import token_logprob
    x = torch.randn(3, 32, device="cuda", requires_grad=True)
    for y in (layer_norm(x), token_logprob(x, torch.zeros(3, dtype=torch.int64, device="cuda"))):
        (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            g.sum().backward()


def test_saved_operand_changed_in_place_is_noticed(cuda_device):
    from cases.preference_loss.op import preference_loss
    x = torch.randn(2, 3, 40, device="cuda", requires_grad=True)
    y = x * 1.0
    loss, _ = preference_loss(y, torch.zeros(2, 3, dtype=torch.int64, device="cuda"),
                              torch.zeros(2, 3, device="cuda"))
    with torch.no_grad():
        y.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_step_captured_in_a_graph(cuda_device):
    """Forward and backward of a whole step captured (fresh leaves, warmed up on a side stream) and
    replayed on new data."""
    from cases.layernorm.op import layer_norm
    from cases.policy_loss.op import policy_loss
    s = inputs(4, 16, 64, 800, 9)
    zero = torch.zeros(4, 16, device="cuda")
    static = torch.zeros_like(s["hidden"]).requires_grad_(True)
    w = s["weight"].clone().requires_grad_(True)

    def run(x):
        logits = layer_norm(x, w, s["bias"], 1e-5) @ s["head"].T
        loss, kl = policy_loss(logits, s["labels"], zero - 4, zero - 4, s["advantage"], kl_coef=0.1)
        return (loss.detach(), kl) + torch.autograd.grad(loss, (x, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static)
    with torch.no_grad():
        static.copy_(s["hidden"])
    graph.replay()
    torch.cuda.synchronize()
    x = s["hidden"].clone().requires_grad_(True)
    for a, b in zip(out, run(x)):
        # The projections run in a library whose choice may differ: fp32 rounding, not bits.
        assert float((a - b).abs().max()) <= 1000 * U32 * (1e-3 + float(b.abs().max()))
