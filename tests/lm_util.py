"""Helpers of the language-model operators' tests: comparison with a 64-bit result."""
import torch

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U32 = 2.0 ** -24  # half a unit in the last place of fp32, relative


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(name, got, want, bound):
    """|got - want| <= bound everywhere; NaN and infinities agree exactly."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).detach().cpu().expand_as(want)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN differ"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{name}: infinities differ"
    err = (got - want).abs()[~odd]
    over = err - bound[~odd]
    if over.numel() and not bool((over <= 0).all()):
        i = int(over.argmax())
        raise AssertionError(f"{name}: error {float(err[i]):.3e} over the bound "
                             f"{float(bound[~odd][i]):.3e} (value {float(want[~odd][i]):.6e}); "
                             f"{int((over > 0).sum())} of {over.numel()} outside")


def rounded(want, dtype):
    """Half a unit of ``dtype`` at ``want`` (its smallest subnormal at least): the error of
    rounding once, taken at a value up to 1% larger for what is added before the rounding."""
    tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
    return 1.01 * half_ulp(dtype) * want.double().abs() + tiny[dtype]
