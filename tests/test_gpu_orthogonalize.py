"""The orthogonalised update on the GPU against the iteration in 64 bits.

The bound comes from a noisy copy of the 64-bit iteration: every operand of a product is off by up
to 2^-21 of itself (22 kept bits and the rounding of what was stored) and every entry of a product
by up to 2^-21 of the product of its row's and column's norms (fp32 accumulation of long sums).
The noise goes through the same iteration, so the bound follows an update's own conditioning.  The
kernel's errors are of this kind and size but not the same draw: a factor 4 for the whole (2-norm)
and 40 for a single entry against the noise's root mean square.

Results of 16 bits are summed in longer runs (1024 deep for fp16, 2048 for bf16) in an accumulator that
truncates: each of the up to 3 MMAs for 16 terms takes up to one unit, 2^-23 of the accumulator, half of
it on average.  The accumulator is at most the product of the norms, so a product of depth K carries up to
3 min(K, run) / 16 * 2^-24 of that: 1.7e-5 at K = 1500 in bf16, 1/200 of its rounding.
"""
import math

import pytest
import torch

from lm_util import DTYPES, half_ulp

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
NOISE = 2.0 ** -21


def iterate(g, steps, coef, eps, noise=None):
    """The iteration in fp64; ``noise``: a generator for the perturbed copy."""
    run = {torch.float32: 0, torch.float16: 1024, torch.bfloat16: 2048}.get(g.dtype, 0)
    coef = [coef] * steps if not isinstance(coef[0], (tuple, list)) else coef
    x = g.double()
    tall = x.size(-2) > x.size(-1)
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)

    def rough(t):
        if noise is None:
            return t
        return t * (1 + NOISE * (2 * torch.rand(t.shape, device=t.device, dtype=t.dtype,
                                                generator=noise) - 1))

    def mul(p, q):
        out = rough(p) @ rough(q)
        if noise is not None:
            size = p.norm(dim=-1, keepdim=True) * q.norm(dim=-2, keepdim=True)
            sums = max(NOISE, 3 * min(p.size(-1), run) / 16 * 2.0 ** -24)
            out = out + sums * size * (2 * torch.rand(out.shape, device=out.device,
                                                       dtype=out.dtype, generator=noise) - 1)
        return out

    for a, b, c in coef:
        k = mul(x, x.mT)
        x = rough(a * x) + mul(b * k + c * mul(k, k), x)
    return x.mT if tall else x


def update(shape, dtype, seed, scale=1e-3):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=g)

    *lead, m, n = shape
    k = min(m, n, 8)
    u = (randn(*lead, m, k) / torch.arange(1, k + 1, device="cuda")) @ randn(*lead, k, n)
    return (scale * (u + 0.5 * randn(*lead, m, n))).to(dtype)


def check(g, steps=5, coef=COEF, eps=EPS, got=None):
    from cases.orthogonalize.op import orthogonalize
    got = orthogonalize(g, steps, coef, eps) if got is None else got
    assert got.shape == g.shape and got.dtype == g.dtype and got.is_contiguous()
    want = iterate(g, steps, coef, eps)
    noisy = iterate(g, steps, coef, eps, torch.Generator(device="cuda").manual_seed(1))
    # What lies beyond the type's range rounds to infinity.
    big = want.abs() > torch.finfo(g.dtype).max * (1 + 2 * half_ulp(g.dtype))
    assert torch.equal(got.double()[big], want[big].sign() * math.inf)
    err = torch.where(big, 0.0, got.double() - want)
    off = noisy - want
    want = torch.where(big, 0.0, want)
    ulp = half_ulp(g.dtype)
    dims = (-2, -1)
    tiny = 2.0 ** -24 if g.dtype == torch.float16 else 0.0
    n = math.sqrt(want.size(-1) * want.size(-2))
    bound = 4 * off.norm(dim=dims) + ulp * want.norm(dim=dims) + (tiny + 1e-9) * n
    assert bool((err.norm(dim=dims) <= bound).all()), (err.norm(dim=dims), bound)
    rms = off.norm(dim=dims, keepdim=True) / n
    entry = 40 * rms + 1.01 * ulp * want.abs() + tiny + 1e-9
    assert bool((err.abs() <= entry).all()), float((err.abs() - entry).max())
    return got


SHAPES = [(1, 1), (1, 9), (9, 1), (2, 3), (16, 16), (31, 33), (64, 64), (65, 63), (100, 300),
          (128, 128), (129, 257), (300, 100), (256, 512), (511, 513), (1000, 1000), (1001, 260),
          (260, 2601), (640, 1920), (2048, 1024), (2000, 2300)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_64_bits(shape, dtype, cuda_device):
    check(update(shape, dtype, shape[0] + shape[1]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(4090, 8190), (8190, 4093), (4100, 8190)])
def test_widest_tiles(shape, dtype, cuda_device):
    """Large enough for tiles of 256 x 256 (the last: x 128), of sizes that fill none."""
    check(update(shape, dtype, 5))


@pytest.mark.parametrize("shape", [(3, 40, 70), (2, 3, 130, 65), (5, 256, 256), (20, 7, 129),
                                   (2, 700, 900), (7, 384, 128)])
def test_batches(shape, cuda_device):
    """Each matrix of a batch is normalised by its own norm."""
    g = update(shape, torch.float32, 3)
    g = g * torch.logspace(-2, 2, shape[0], device="cuda").view(-1, *[1] * (g.dim() - 1))
    got = check(g)
    from cases.orthogonalize.op import orthogonalize
    one = orthogonalize(g[1])
    # Another tile split may be chosen for the single matrix: equal within the noise.
    assert float((one - got[1]).abs().max()) < 1e-3


def test_singular_values_end_near_one(cuda_device):
    g = torch.randn(300, 500, device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    s = torch.linalg.svdvals(check(g).double())
    assert float(s.max()) < 1.25 and float(s.min()) > 0.3


@pytest.mark.parametrize("steps", [1, 2, 7])
def test_steps_and_schedules(steps, cuda_device):
    g = update((150, 220), torch.float32, 9)
    check(g, steps)
    other = [(3.0, -3.2, 1.2), (1.875, -1.25, 0.375)]  # the second: a plain quintic iteration
    check(g, steps, [other[min(k, 1)] for k in range(steps)])
    check(g, steps, (1.5, -0.5, 0.0))  # cubic


def test_ill_conditioned(cuda_device):
    """Singular values over eight decades: those far below 1/500 stay small, none blow up."""
    g = torch.Generator("cuda").manual_seed(2)
    q1 = torch.linalg.qr(torch.randn(200, 200, device="cuda", dtype=torch.float64, generator=g))[0]
    q2 = torch.linalg.qr(torch.randn(350, 200, device="cuda", dtype=torch.float64, generator=g))[0]
    s = torch.logspace(0, -8, 200, device="cuda", dtype=torch.float64)
    check(((q1 * s) @ q2.T).float())


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1.0, 1e15])
def test_magnitudes(scale, cuda_device):
    """Any magnitude (eps = 0); with the default eps a tiny update stays tiny."""
    g = update((90, 140), torch.float32, 4, scale)
    check(g, eps=0.0)
    got, want = check(g) if scale >= 1e-3 else None, iterate(g, 5, COEF, EPS)
    if got is None:
        from cases.orthogonalize.op import orthogonalize
        got = orthogonalize(g).double()
        assert float((got - want).norm()) <= 1e-5 * float(want.norm())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("share", [0.1, 0.5, 0.99, 1.01, 3.0])
def test_norm_near_eps(share, dtype, cuda_device):
    """eps of a share of the update's norm: the first X is well below 1."""
    g = update((130, 300), dtype, 8)
    check(g, eps=share * float(g.double().norm()))


def test_zero_and_nan(cuda_device):
    from cases.orthogonalize.op import orthogonalize
    g = update((3, 50, 60), torch.float32, 6)
    g[1] = 0
    g[2, 4, 5] = float("nan")
    out = orthogonalize(g)
    assert torch.isfinite(out[0]).all() and not out[1].any() and torch.isnan(out[2]).all()
    assert torch.isnan(orthogonalize(torch.zeros(4, 5, device="cuda"), eps=0.0)).all()


def test_diverging_coefficients_do_not_fault(cuda_device):
    from cases.orthogonalize.op import orthogonalize
    g = update((70, 80), torch.float32, 7)
    out = orthogonalize(g, 6, (30.0, 20.0, 10.0))
    assert not torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_updates(dtype, cuda_device):
    base = update((4, 200, 330), dtype, 8)
    for v in (base[:, :, :150], base[:, 3:, 5:200], base[1].t(), base.transpose(1, 2), base[::2],
              base[2, :, ::3], base[0:1].expand(3, 200, 330), base.view(2, 2, 200, 330)[:, 1]):
        check(v.contiguous(), got=__import__("cases.orthogonalize.op", fromlist=["x"]).orthogonalize(
            v, 5, COEF, EPS))


def test_equal_calls_and_streams(cuda_device):
    from cases.orthogonalize.op import orthogonalize
    g = update((2, 300, 500), torch.bfloat16, 10)
    want = orthogonalize(g)
    assert torch.equal(orthogonalize(g), want)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s1):
        a = orthogonalize(g)
    with torch.cuda.stream(s2):
        b = orthogonalize(g)
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)


def test_captured_and_replayed_on_new_data(cuda_device):
    from cases.orthogonalize.op import orthogonalize
    g = update((300, 260), torch.bfloat16, 11)
    want = orthogonalize(g)
    static = torch.zeros_like(g)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = orthogonalize(static)
        graphs.append((graph, out))
    static.copy_(g)
    for graph, out in graphs * 2:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_wait_that_runs_out_is_reported(cuda_device, monkeypatch):
    from cases.orthogonalize.op import orthogonalize
    g = update((200, 200), torch.float32, 12)
    monkeypatch.setenv("RBF_CHECK_STATUS", "1")
    want = orthogonalize(g, 1)
    monkeypatch.setenv("RBF_DEBUG_SKIP_FIRST_LOAD", "1")
    monkeypatch.setenv("RBF_WAIT_TIMEOUT_MS", "20")
    with pytest.raises(RuntimeError, match="status 7"):
        orthogonalize(g, 1)
    monkeypatch.delenv("RBF_DEBUG_SKIP_FIRST_LOAD")
    monkeypatch.delenv("RBF_WAIT_TIMEOUT_MS")
    assert torch.equal(orthogonalize(g, 1), want)


def test_empty_and_refusals(cuda_device):
    from cases.orthogonalize.op import orthogonalize
    assert orthogonalize(torch.empty(0, 5, device="cuda")).shape == (0, 5)
    assert orthogonalize(torch.empty(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    x = torch.randn(4, 5, device="cuda")
    with pytest.raises(RuntimeError, match="steps"):
        orthogonalize(x, steps=33)
    with pytest.raises(RuntimeError, match="eps"):
        orthogonalize(x, eps=-1.0)
    with pytest.raises(RuntimeError, match="coefficient"):
        orthogonalize(x, coefficients=(1.0, float("nan"), 0.0))
    with pytest.raises(RuntimeError, match="gradient"):
        orthogonalize(x.requires_grad_(True))


def test_verify_all_passes(cuda_device):
    from cases.orthogonalize import CASE
    from cases.orthogonalize.op import candidate
    from framework.verify import verify_all
    ok, report = verify_all(CASE, candidate, device="cuda")
    assert ok and "[backward] none" in report, report


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(40, 400), (129, 1300), (1500, 300), (3, 70, 500), (20, 200, 1500), (8000, 300)])
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 8])
def test_groups_of_steps(shape, steps, dtype, cuda_device):
    """Long rows: 16-bit types take several steps through X at once, of every group size, with
    coefficients that change from step to step and with some that forbid a group."""
    g = update(shape, dtype, sum(shape) + steps)
    check(g, steps)
    schedule = [(3.4445, -4.775, 2.0315), (3.0, -3.2, 1.2), (2.5, -2.0, 0.6), (1.875, -1.25, 0.375)]
    check(g, steps, [schedule[k % 4] for k in range(steps)])
    # a^2 = 225 is past what a group may carry: these two steps (15 times, then back) stand alone.
    check(g, steps, ([(15.0, 0.0, 0.0), (1 / 15, 0.0, 0.0)] + [(1.875, -1.25, 0.375)] * steps)[:steps])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (8, 64), (3, 40, 70), (4, 256, 256), (300, 1100), (2100, 1001)])
def test_equal_calls_give_equal_bits(shape, dtype, cuda_device, monkeypatch):
    """Calls back to back, every other one with another update (and so other contents in the workspace that
    the next one gets): each product reads what this call's products wrote, and CTA pairs that end at
    once leave no arrival behind for the next call."""
    from cases.orthogonalize.op import orthogonalize
    g, other = update(shape, dtype, sum(shape)), update(shape, dtype, 1 + sum(shape), scale=30.0)
    want = orthogonalize(g)
    torch.cuda.synchronize()
    outs = []
    for _ in range(60):
        orthogonalize(other)
        outs.append(orthogonalize(g))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)
    monkeypatch.setenv("RBF_CHECK_STATUS", "1")
    assert torch.equal(orthogonalize(g), want)


@pytest.mark.parametrize("shape", [(60, 60), (2, 120, 834), (3, 131, 512), (6, 555, 133), (2, 194, 81), (3574, 320), (6, 365, 1135),
                                   (6, 111, 3322), (130, 4000), (512, 512), (700, 4096), (2601, 1001), (1100, 2800)])
def test_fp32_is_as_exact_as_fp32_products(shape, cuda_device):
    """Against the iteration in 64 bits, the error (Frobenius norm) is at most half again what the same iteration in
    fp32 products has: operands of 22 bits and truncated sums cost no more than that."""
    from cases.orthogonalize.op import orthogonalize
    gen = torch.Generator(device="cuda").manual_seed(sum(shape))
    batch = shape if len(shape) == 3 else (1, *shape)
    b, m, n = batch
    fall = 1.0 / torch.arange(1, 17, device="cuda")
    strong = (torch.randn(b, m, 16, device="cuda", generator=gen) * fall) @ torch.randn(b, 16, n, device="cuda", generator=gen)
    g = (1e-3 * (strong + 0.5 * torch.randn(b, m, n, device="cuda", generator=gen))).view(shape)
    want = iterate(g, 5, COEF, EPS)
    x = g.mT if m > n else g
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(5):
        k = x @ x.mT
        x = COEF[0] * x + (COEF[1] * k + COEF[2] * (k @ k)) @ x
    plain = x.mT if m > n else x

    def error(t):
        return float((t.double() - want).norm() / want.norm())

    got = error(orthogonalize(g))
    assert got <= 1.5 * error(plain), (got, error(plain))


def test_status_is_not_read_inside_a_capture(cuda_device, monkeypatch):
    from cases.orthogonalize.op import orthogonalize
    monkeypatch.setenv("RBF_CHECK_STATUS", "1")
    g = update((100, 300), torch.bfloat16, 4)
    want = orthogonalize(g)
    static = torch.zeros_like(g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(static)
    static.copy_(g)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
