"""The language-model operators on the CPU: the library exports what include/lm_sm100.h declares,
its entries and the Python calls refuse bad arguments before they touch a device, and the cases'
definitions match independent formulas and finite differences."""
import importlib
import math
import os
import re

import pytest
import torch

import lm_abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, MISALIGNED, WORKSPACE, UNSUPPORTED = 0, 1, 2, 3, 4
A = 1 << 20  # an aligned address that is never touched: every refusal comes first


@pytest.fixture(scope="module")
def lib():
    return lm_abi.lib()


def test_library_exports_the_header(lib):
    text = open(os.path.join(ROOT, "include", "lm_sm100.h")).read()
    names = re.findall(r"RBF_API\s+\w+\s+(\w+)\s*\(", text)
    assert len(names) >= 8
    assert set(names) == set(lm_abi.SIGNATURES)
    assert all(hasattr(lib, n) for n in names)


def ln_forward(lib, x=A, stride=8, w=A, b=A, y=A, mean=A, rstd=A, rows=4, D=8, eps=1e-5, dt=0,
               wdt=0):
    return lib.ln_sm100_forward(x, stride, w, b, y, mean, rstd, rows, D, eps, dt, wdt, None)


def test_layernorm_refusals(lib):
    assert ln_forward(lib, rows=-1) == INVALID
    assert ln_forward(lib, D=1 << 31, stride=1 << 31) == UNSUPPORTED
    assert ln_forward(lib, stride=7) == INVALID
    assert ln_forward(lib, eps=-1.0) == INVALID
    assert ln_forward(lib, eps=math.nan) == INVALID
    assert ln_forward(lib, dt=3) == INVALID
    assert ln_forward(lib, x=None) == INVALID
    assert ln_forward(lib, x=A + 2) == MISALIGNED
    assert ln_forward(lib, y=A + 1, dt=1) == MISALIGNED
    assert ln_forward(lib, w=A + 2) == MISALIGNED
    assert ln_forward(lib, mean=None) == INVALID
    assert b"mean" in lib.rbf_sm100_last_error_detail()
    need = lib.ln_sm100_backward_workspace_bytes(4, 8)
    assert need >= 2 * 4 * 8 and lib.ln_sm100_backward_workspace_bytes(-1, 8) == 0

    def back(dy=A, x=A, stride=8, mean=A, dx=A, dw=A, ws=A, size=need):
        return lib.ln_sm100_backward(dy, 8, x, stride, A, mean, A, dx, dw, None, 4, 8, 0, 0, ws,
                                     size, None)
    assert back(dy=None) == INVALID
    assert back(stride=3) == INVALID
    assert back(mean=None) == INVALID
    assert back(size=need - 1) == WORKSPACE
    assert back(ws=None) == WORKSPACE
    assert back(ws=A + 8) == MISALIGNED
    assert back(dx=None, dw=None, ws=None, size=0) == OK  # nothing asked for: nothing launched


def test_logprob_refusals(lib):
    def fwd(x=A, sb=40, st=8, lab=A, lp=A, rows=10, T=5, V=8, dt=0):
        return lib.lp_sm100_forward(x, sb, st, lab, lp, None, None, rows, T, V, -100, dt, None)
    assert fwd(rows=-1) == INVALID
    assert fwd(rows=1 << 61, T=1) == UNSUPPORTED  # 8 times that passes 64 bits
    assert fwd(T=4) == INVALID
    assert fwd(T=0) == INVALID
    assert fwd(V=0) == INVALID
    assert fwd(V=1 << 31) == UNSUPPORTED
    assert fwd(sb=-1) == INVALID
    assert fwd(dt=7) == INVALID
    assert fwd(x=None) == INVALID
    assert fwd(x=A + 2) == MISALIGNED
    assert fwd(lab=A + 4) == MISALIGNED
    assert fwd(lp=None) == INVALID

    def bwd(stats=A, coef=A, s0=None, dx=A, rows=10, V=8):
        return lib.lp_sm100_backward(A, 40, 8, A, stats, coef, s0, None, dx, rows, 5, V, -100, 0,
                                     None)
    assert bwd(stats=None) == INVALID
    assert bwd(coef=A + 1) == MISALIGNED
    assert bwd(s0=A + 2) == MISALIGNED
    assert bwd(dx=None) == INVALID
    assert bwd(rows=5 << 26) == UNSUPPORTED


def test_loss_refusals(lib):
    size = lib.loss_sm100_workspace_bytes(4, 10)
    assert size >= 3 * 8 * 4

    def pref(B=4, T=10, beta=0.1, s=0.0, lp=A, loss=A, ws=A, n=size):
        return lib.pref_sm100_loss(lp, None, A, A, loss, A, A, B, T, beta, s, -100, ws, n, None)
    assert pref(B=3) == INVALID
    assert pref(B=-2) == INVALID
    assert pref(beta=math.inf) == INVALID
    assert pref(s=1.5) == INVALID and pref(s=math.nan) == INVALID
    assert pref(lp=None) == INVALID
    assert pref(loss=None) == INVALID
    assert pref(n=size - 1) == WORKSPACE

    def pol(lo=0.2, hi=0.2, k=0.0, adv=A, norm=A, ws=A, n=size):
        return lib.policy_sm100_loss(A, None, A, A, adv, 0, A, A, A, A, norm, 4, 10, lo, hi, k, -100, ws,
                                     n, None)
    assert pol(lo=-0.1) == INVALID and pol(hi=math.nan) == INVALID
    assert pol(k=math.nan) == INVALID
    assert pol(adv=None) == INVALID
    assert pol(norm=None) == INVALID
    assert pol(ws=None) == WORKSPACE


def test_python_calls_refuse_cpu_tensors_and_bad_types():
    from cases.layernorm.op import layer_norm
    from cases.policy_loss.op import policy_loss
    from cases.preference_loss.op import preference_loss
    from cases.token_logprob.op import token_logprob
    x, lab = torch.randn(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64)
    z = torch.zeros(2, 3)
    for call in (lambda: layer_norm(x), lambda: token_logprob(x, lab),
                 lambda: preference_loss(x, lab, z),
                 lambda: policy_loss(x, lab, z, z, torch.ones(2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


NAMES = ["layernorm", "token_logprob", "preference_loss", "policy_loss"]


@pytest.mark.parametrize("name", NAMES)
def test_case_surface(name, monkeypatch):
    mod = importlib.import_module(f"cases.{name}")
    assert mod.CASE.name == name and mod.CASE.description.startswith("#")
    assert set(mod.CASE.grad_inputs) <= {"x", "weight", "bias", "logits"}
    config = importlib.import_module(f"cases.{name}.config")
    for k, v in {"ROWS": 6, "D": 10, "B": 4, "T": 5, "V": 30}.items():
        if hasattr(config, k):
            monkeypatch.setattr(config, k, v)
    a = mod.CASE.make_inputs(3, torch.float32, "cpu", requires_grad=True)
    b = mod.CASE.make_inputs(3, torch.float32, "cpu")
    assert all(torch.equal(a[k], b[k]) for k in a)
    out = mod.CASE.reference_forward(a, mod.CASE.params)
    out.sum().backward()
    assert all(a[k].grad is not None for k in mod.CASE.grad_inputs)


def test_layernorm_definition():
    from cases.layernorm.reference import reference_forward
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((4, 9), (9,), (9,)))
    got = reference_forward({"x": x, "weight": w, "bias": b}, {"eps": 1e-5})
    want = torch.nn.functional.layer_norm(x, (9,), w, b, 1e-5)
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-12)


def test_loss_definitions():
    from cases.policy_loss.reference import policy
    from cases.preference_loss.reference import preference
    from cases.token_logprob.reference import logprob
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 6, 11, generator=g, dtype=torch.float64)
    lab = torch.randint(0, 11, (4, 6), generator=g)
    lab[0, :2] = -100
    lp = logprob(x, lab, -100)
    want = torch.nn.functional.cross_entropy(x.reshape(-1, 11), lab.reshape(-1),
                                             ignore_index=-100, reduction="none")
    torch.testing.assert_close(lp.reshape(-1), -want, rtol=1e-12, atol=1e-12)
    ref = lp.float() + 0.1
    loss, reward = preference(lp, ref, lab, 0.5, 0.0, -100)
    by_hand = 0.0
    for p in range(2):
        m = lab != -100
        r = [0.5 * sum(float(lp[i, t]) - float(ref[i, t]) for t in range(6) if m[i, t])
             for i in (p, p + 2)]
        by_hand += math.log(1 + math.exp(-(r[0] - r[1]))) / 2
    assert abs(float(loss) - by_hand) < 1e-9
    old, adv = (lp - 0.3).float(), torch.tensor([1.0, -1.0, 2.0, 0.5])
    loss, kl = policy(lp, old, ref, adv, lab, 0.2, 0.2, 0.1, -100)
    total = n = 0.0
    for i in range(4):
        for t in range(6):
            if lab[i, t] == -100:
                continue
            r = math.exp(float(lp[i, t]) - float(old[i, t]))
            d = float(ref[i, t]) - float(lp[i, t])
            a = float(adv[i])
            total += 0.1 * (math.exp(d) - d - 1) - min(r * a, min(max(r, 0.8), 1.2) * a)
            n += 1
    assert abs(float(loss) - total / n) < 1e-9 and float(kl) > 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_layernorm_reference_rounds_once(dtype, monkeypatch):
    """An exact implementation, 64 bits and one rounding, passes the gate in every type that the case offers."""
    import dataclasses

    from cases.layernorm import CASE, config
    from framework.verify import verify_all
    monkeypatch.setattr(config, "ROWS", 512)
    monkeypatch.setattr(config, "D", 256)

    def exact(inputs, params):
        x, w, b = (inputs[k].double() for k in ("x", "weight", "bias"))
        y = torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, params["eps"])
        return y.to(inputs["x"].dtype)

    ok, report = verify_all(dataclasses.replace(CASE, dtype=dtype), exact, device="cpu")
    assert ok, report
