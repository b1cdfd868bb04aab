"""The verify and bench harness on the language-model cases, in every type that they offer."""
import dataclasses
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = ["layernorm", "token_logprob", "preference_loss", "policy_loss", "orthogonalize"]


def load(name):
    return (importlib.import_module(f"cases.{name}").CASE,
            importlib.import_module(f"cases.{name}.op"))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("name", CASES)
def test_verify_all_passes_in_16_bits(name, dtype, cuda_device):
    from framework.verify import verify_all
    case, op = load(name)
    ok, report = verify_all(dataclasses.replace(case, dtype=dtype), op.candidate, device="cuda")
    assert ok, report


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", CASES)
def test_bench_compare_times_the_case(name, dtype, cuda_device, monkeypatch):
    """framework/bench.py's run over a case: both passes timed, or the one there is."""
    from framework import bench
    case, op = load(name)
    monkeypatch.setattr(bench, "PROTOCOL", dataclasses.replace(
        bench.PROTOCOL, warmup=1, iters=3, repeats=2, max_retries=0))
    report, _ = bench.compare(dataclasses.replace(case, dtype=dtype), op.candidate, device="cuda",
                              baseline=case.reference_forward)
    assert "[candidate]" in report and "gate:" in report
    assert report.count("backward:") == (3 if case.grad_inputs else 0), report


@pytest.mark.parametrize("name", CASES)
def test_forward_only_is_the_candidates_forward(name, cuda_device):
    case, op = load(name)
    inputs = case.make_inputs(0, torch.float32, cuda_device)
    with torch.no_grad():
        assert torch.equal(op.forward_only(inputs, case.params), op.candidate(inputs, case.params))
