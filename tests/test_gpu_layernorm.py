"""Layer norm on the GPU against a 64-bit implementation of its formulas."""
import pytest
import torch

from lm_util import DTYPES, U32, assert_within, rounded

pytestmark = pytest.mark.gpu

EPS = 1e-5


def inputs(rows, D, dtype, wdtype, seed, offset=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, device="cuda", generator=g)

    x = (randn(rows, D) * 2 + offset).to(dtype)
    return x, (1 + 0.3 * randn(D)).to(wdtype), (0.2 * randn(D)).to(wdtype), randn(rows, D).to(dtype)


def formulas(x, w, b, dy, eps):
    """(y, dx, dw, db, rstd) in fp64."""
    x, dy = x.double(), dy.double()
    D = x.size(1)
    w = torch.ones(D, device=x.device).double() if w is None else w.double()
    b = torch.zeros(D, device=x.device).double() if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    h = (x - mean) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return h * w + b, dx, (dy * h).sum(0), dy.sum(0), rstd


def bounds(x, w, b, dy, want, dtype, wdtype):
    """Errors of the fp32 arithmetic plus one rounding of each output.

    A row's sums add at most 16 values in a lane and 10 levels of lanes and warps: 26 roundings,
    each of at most U32 of the sum of absolute values.  So mean is off by 26 U32 mean|x| plus the
    division, xh by that times rstd plus a few roundings of xh itself (the variance's relative
    error halves in rstd): within e = 40 U32 (max|x| rstd + |xh|).  g's sums are off by 26 U32 of
    mean|g| and of mean|g xh|, plus e times mean|g|.  Columns: every addend carries e, and the
    sum of n rows at most (rows + 32) U32 of the absolute sum (a running sum, then a tree)."""
    y, dx, dw, db, rstd = want
    xd, dyd = x.double(), dy.double()
    wd = torch.ones_like(xd[0]) if w is None else w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    h = (xd - xd.mean(1, keepdim=True)) * rstd
    e = 40 * U32 * (xd.abs().amax(1, keepdim=True) * rstd + h.abs())
    g = dyd * wd
    gm = g.abs().mean(1, keepdim=True)
    gh = (g * h).abs().mean(1, keepdim=True)
    hm = (h * h).mean(1, keepdim=True).sqrt()
    eg = 30 * U32 * (g.abs() + gm)
    eh = e * gh + h.abs() * ((g.abs() * e).mean(1, keepdim=True) + 30 * U32 * (gh + gm * hm))
    n = x.size(0)
    return {
        "y": e * wd.abs() + 3 * U32 * (h * wd).abs() + 2 * U32 * bd.abs() + rounded(y, dtype),
        "dx": rstd * (eg + eh) + 30 * U32 * dx.abs() + rounded(dx, dtype),
        "dw": (dyd.abs() * e).sum(0) + (n + 32) * U32 * (dyd * h).abs().sum(0) + rounded(dw, wdtype),
        "db": (n + 32) * U32 * dyd.abs().sum(0) + rounded(db, wdtype),
    }


def check(x, w, b, dy, eps=EPS):
    from cases.layernorm.op import layer_norm
    wdtype = w.dtype if w is not None else b.dtype if b is not None else x.dtype
    want = formulas(x, w, b, dy, eps)
    bound = bounds(x, w, b, dy, want, x.dtype, wdtype)
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    y.backward(dy)
    assert y.dtype == x.dtype
    assert_within("y", y, want[0], bound["y"])
    assert_within("dx", leaves[0].grad, want[1], bound["dx"])
    if w is not None:
        assert_within("dw", leaves[1].grad, want[2], bound["dw"])
    if b is not None:
        assert_within("db", leaves[2].grad, want[3], bound["db"])
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps), y.detach())


SHAPES = [(1, 1), (3, 2), (1, 48), (8, 64), (5, 127), (300, 128), (33, 255), (7, 256), (9, 257),
          (40, 511), (40, 512), (600, 513), (3, 1000), (64, 1023), (65, 1024), (2, 2048),
          (17, 4095), (513, 4096), (4, 6000), (3, 8192), (5, 8194), (2, 16383), (3, 16384),
          (2, 16385), (5, 40000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", SHAPES)
def test_against_formulas(rows, D, dtype, cuda_device):
    check(*inputs(rows, D, dtype, dtype, rows * 31 + D))


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("rows,D", [(9, 130), (50, 1024), (3, 16384), (2, 20000)])
def test_fp32_parameters(rows, D, dtype, cuda_device):
    check(*inputs(rows, D, dtype, torch.float32, D))


@pytest.mark.parametrize("has_w,has_b", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("D", [96, 4096, 17000])
def test_without_parameters(has_w, has_b, D, cuda_device):
    x, w, b, dy = inputs(6, D, torch.bfloat16, torch.bfloat16, D)
    check(x, w if has_w else None, b if has_b else None, dy)


def test_large_offset_does_not_cancel(cuda_device):
    """mean 1000 times the deviation: the two-pass variance keeps its digits (the bound scales
    with max|x| rstd, a one-pass E[x^2] - mean^2 would be off by its square)."""
    x, w, b, dy = inputs(20, 3000, torch.float32, torch.float32, 5, offset=2000.0)
    check(x, w, b, dy)


@pytest.mark.parametrize("rows,D", [(1000, 64), (40000, 136)])
def test_many_rows(rows, D, cuda_device):
    check(*inputs(rows, D, torch.float32, torch.float32, 77))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", [(310, 9001), (200, 12290), (200, 12292), (330, 6004), (333, 16376)])
def test_many_long_rows(rows, D, dtype, cuda_device):
    """More long rows than CTAs, at every alignment."""
    check(*inputs(rows, D, dtype, dtype, D))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", [(64, 1), (65, 7), (71, 31), (64, 255), (4099, 1023), (2100, 1001), (1200, 2041), (1200, 2042),
                                    (700, 4085), (700, 4089), (700, 4090), (530, 4094), (20000, 129), (530, 4095), (520, 8185), (520, 8189), (260, 16377),
                                    (260, 16378)])
def test_unaligned_rows(rows, D, dtype, cuda_device):
    """Rows that begin anywhere in 16 bytes, at the ends of what a CTA's threads hold."""
    check(*inputs(rows, D, dtype, dtype, D))


@pytest.mark.parametrize("dtype", DTYPES)
def test_unaligned_rows_apart(dtype, cuda_device):
    """Rows with gaps that shift like contiguous ones, or not; a first row off 16 bytes; nothing of the gaps
    (NaN) reaches a result."""
    x, w, b, dy = inputs(900, 2600 + 3, dtype, dtype, 3)
    for gap, first in ((8, 0), (16, 0), (5, 0), (8, 8), (8, 3)):
        big = torch.full((900, 2603 + gap), float("nan"), dtype=dtype, device=x.device)
        wide = big.reshape(-1)[first:first + 899 * (2603 + gap) + 2603].as_strided((900, 2603), (2603 + gap, 1))
        wide.copy_(x)
        check(wide, w, b, dy)
        check(x, w, None, wide)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", [(5, 512), (100, 512), (2100, 1024), (70, 6144), (70, 12288)])
def test_misaligned_parameters(rows, D, dtype, cuda_device):
    """Weight and bias that begin off 16 bytes, under rows that do not."""
    x, w, b, dy = inputs(rows, D, dtype, torch.float32, D)
    for pdtype in {dtype, torch.float32}:
        both = torch.zeros(2 * D + 3, dtype=pdtype, device=x.device)
        both[1:D + 1], both[D + 2:2 * D + 2] = w, b
        check(x, both[1:D + 1], both[D + 2:2 * D + 2], dy)


def test_strided_and_broadcast_operands(cuda_device):
    """Rows that lie apart, a transposed matrix, a misaligned slice, an expanded dy."""
    from cases.layernorm.op import layer_norm
    base, w, b, _ = inputs(60, 512, torch.bfloat16, torch.bfloat16, 3)
    views = [base[:, :256], base[:, 3:259], base[::2, 8:264], base.t()[:256].t(),
             base.view(12, 5, 512)[:, :, 100:356], base.view(12, 5, 512)[:, 2:4, :256]]
    for v in views:
        x = v.detach().requires_grad_(True)
        ww, bb = (t[:256].detach().requires_grad_(True) for t in (w, b))
        dy = torch.full((), 0.5, dtype=x.dtype, device="cuda").expand(x.shape)
        y = layer_norm(x, ww, bb, EPS)
        y.backward(dy)
        flat = v.reshape(-1, 256).contiguous()
        full = dy.reshape(-1, 256).contiguous()
        want = formulas(flat, ww.detach(), bb.detach(), full, EPS)
        bound = bounds(flat, ww.detach(), bb.detach(), full, want, x.dtype, x.dtype)
        assert_within("y", y.reshape(-1, 256), want[0], bound["y"])
        assert_within("dx", x.grad.reshape(-1, 256), want[1], bound["dx"])
        assert_within("dw", ww.grad, want[2], bound["dw"])
        assert_within("db", bb.grad, want[3], bound["db"])


def test_empty_operands(cuda_device):
    from cases.layernorm.op import layer_norm
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = layer_norm(x, w, None, EPS)
    y.sum().backward()
    assert y.shape == (0, 64) and x.grad.shape == (0, 64)
    assert torch.equal(w.grad, torch.zeros_like(w))
    assert layer_norm(torch.empty(4, 0, device="cuda")).shape == (4, 0)


def test_constant_rows_and_nan_stay_in_their_row(cuda_device):
    from cases.layernorm.op import layer_norm
    x, w, b, _ = inputs(8, 300, torch.float32, torch.float32, 9)
    x[2] = 7.0
    x[5, 10] = float("nan")
    y = layer_norm(x, w, b, EPS)
    assert torch.equal(y[2], b)
    assert torch.isnan(y[5]).all()
    assert torch.isfinite(y[[0, 1, 2, 3, 4, 6, 7]]).all()


def test_equal_calls_give_equal_bits(cuda_device):
    from cases.layernorm import native
    x, w, b, dy = inputs(5000, 1000, torch.bfloat16, torch.float32, 1)
    y, stats = native.ln_forward(x, w, b, EPS)
    first = native.ln_backward(dy, x, w, stats)
    for _ in range(3):
        for a, c in zip(first, native.ln_backward(dy, x, w, stats)):
            assert torch.equal(a, c)


def test_gradient_against_differences(cuda_device):
    """The directional derivative of sum(y * dy) by central differences of the fp64 formulas."""
    from cases.layernorm.op import layer_norm
    x, w, b, dy = inputs(6, 70, torch.float32, torch.float32, 21)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    layer_norm(*leaves, EPS).backward(dy)
    g = torch.Generator(device="cuda").manual_seed(4)
    for k in range(3):
        v = torch.randn(leaves[k].shape, device="cuda", generator=g).double()
        h = 1e-5
        def f(s):
            t = [u.detach().double() for u in leaves]
            t[k] = t[k] + s * v
            return float((formulas(*t, dy, EPS)[0] * dy.double()).sum())
        want = (f(h) - f(-h)) / (2 * h)
        got = float((leaves[k].grad.double() * v).sum())
        # h^2 of the third derivative and fp64 cancellation (1e-16 / h) are below 1e-6 here.
        assert abs(got - want) <= 1e-5 * (1 + float((leaves[k].grad.double().abs() * v.abs()).sum()))


def test_other_stream_and_graph(cuda_device):
    """On a side stream, and captured with its backward and replayed on new data."""
    from cases.layernorm import native
    x, w, b, dy = inputs(700, 768, torch.bfloat16, torch.bfloat16, 2)
    want = native.ln_forward(x, w, b, EPS)
    wantb = native.ln_backward(dy, x, w, want[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y, stats = native.ln_forward(x, w, b, EPS)
        out = native.ln_backward(dy, x, w, stats)
    s.synchronize()
    assert torch.equal(y, want[0]) and all(torch.equal(p, q) for p, q in zip(out, wantb))
    sx, sdy = torch.zeros_like(x), torch.zeros_like(dy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, stats = native.ln_forward(sx, w, b, EPS)
        out = native.ln_backward(sdy, sx, w, stats)
    sx.copy_(x)
    sdy.copy_(dy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want[0]) and all(torch.equal(p, q) for p, q in zip(out, wantb))


def test_verify_all_passes(cuda_device):
    from cases.layernorm import CASE
    from cases.layernorm.op import candidate
    from framework.verify import verify_all
    ok, report = verify_all(CASE, candidate, device="cuda")
    assert ok, report


@pytest.mark.parametrize("D", [40, 1000, 1023, 4096, 9000, 20000])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_single_gradient(D, which, cuda_device):
    """Only one of x, weight and bias requires a gradient: it equals the one among all three."""
    from cases.layernorm.op import layer_norm
    x, w, b, dy = inputs(37, D, torch.bfloat16, torch.float32, D + which)
    every = [t.clone().requires_grad_(True) for t in (x, w, b)]
    layer_norm(*every, EPS).backward(dy)
    one = [t.clone().requires_grad_(k == which) for k, t in enumerate((x, w, b))]
    layer_norm(*one, EPS).backward(dy)
    for k in range(3):
        assert (one[k].grad is not None) == (k == which)
    assert torch.equal(one[which].grad, every[which].grad)


def test_offsets_past_32_bits(cuda_device):
    """2^31 values and more: the last rows, and the column sums of rows beyond the boundary."""
    from cases.layernorm import native
    rows, D = (1 << 31) // 4096 + 700, 4096
    x = torch.zeros(rows, D, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros_like(x)
    tail, w, b, up = inputs(600, D, torch.bfloat16, torch.bfloat16, 3)
    x[-600:], dy[-600:] = tail, up
    y, stats = native.ln_forward(x, w, b, EPS)
    ys, ss = native.ln_forward(tail, w, b, EPS)
    assert torch.equal(y[-600:], ys) and torch.equal(y[0], b) and torch.equal(y[-601], b)
    dx, dw, db = native.ln_backward(dy, x, w, stats)
    dxs, dws, dbs = native.ln_backward(up, tail, w, ss)
    assert torch.equal(dx[-600:], dxs) and not dx[:-600].any()
    # The other rows add zeros, in another grouping of the sums: a few fp32 roundings, then one.
    for p, q in ((dw, dws), (db, dbs)):
        assert float((p.float() - q.float()).abs().max()) <= 2.0 ** -7 * float(q.abs().max())


# What adds up a column: a CTA's rows one after another (144 CTAs or more where there are that many rows, blocks
# of up to 4 rows), its groups (16 at most), and the CTAs' partial sums, 32 of them side by side: ten after one
# another, then 32.
def column_chain(rows):
    return -(-rows // 144) + 4 + 16 + 10 + 32


def check_columns(rows, D, dtype, dy, seed):
    """dweight and dbias in fp32 within the roundings of their chain of additions."""
    from cases.layernorm import native
    x, w, b, _ = inputs(rows, D, dtype, torch.float32, seed)
    want = formulas(x, w, b, dy, EPS)
    h = (x.double() - x.double().mean(1, keepdim=True)) * want[4]
    e = 40 * U32 * (x.double().abs().amax(1, keepdim=True) * want[4] + h.abs())  # of h, as in `bounds`
    size = dy.double().abs()
    chain = column_chain(rows) * U32
    _, stats = native.ln_forward(x, w, b, EPS)
    _, dw, db = native.ln_backward(dy, x, w, stats)
    assert_within("dw", dw, want[2], (size * e).sum(0) + chain * (size * h.abs()).sum(0) + rounded(want[2], torch.float32))
    assert_within("db", db, want[3], chain * size.sum(0) + rounded(want[3], torch.float32))


COLUMNS = [(40000, 136), (20000, 129), (4099, 1023), (2100, 1024), (1200, 2041), (530, 4096), (700, 4089), (520, 8189), (310, 9001),
           (330, 6004), (200, 12290), (90, 20000), (60, 100), (33, 1001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", COLUMNS)
def test_column_sums_within_their_chain(rows, D, dtype, cuda_device):
    dy = inputs(rows, D, dtype, dtype, rows + D)[3]
    check_columns(rows, D, dtype, dy, rows + D + 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D", COLUMNS)
def test_every_row_is_in_the_column_sums(rows, D, dtype, cuda_device):
    """dy is 0 but for a few rows: the first and the last ones (every class of alignment, a CTA's last block) and
    some between, so that the bound is a few roundings of those and a row left out shows at its full size."""
    full = inputs(rows, D, dtype, dtype, rows * D)[3]
    gen = torch.Generator().manual_seed(rows)
    for some in (list(range(9)), list(range(rows - 9, rows)), torch.randint(0, rows, (8,), generator=gen).tolist()):
        dy = torch.zeros_like(full)
        dy[some] = full[some]
        check_columns(rows, D, dtype, dy, rows + 3)


@pytest.mark.parametrize("has_w,has_b", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("rows,D", [(2100, 1024), (2100, 1001), (530, 4096), (70, 6004), (70, 12288), (33, 1001), (300, 8188)])
def test_without_parameters_on_every_path(rows, D, has_w, has_b, cuda_device):
    """Rings of whole packs and of shifted rows, rows taken one at a time, long rows."""
    for dtype in (torch.bfloat16, torch.float32):
        x, w, b, dy = inputs(rows, D, dtype, torch.float32, D)
        check(x, w if has_w else None, b if has_b else None, dy)


@pytest.mark.parametrize("rows,D", [(2100, 1024), (2100, 1001), (530, 4096), (70, 12288)])
def test_nan_stays_in_its_row_of_a_block(rows, D, cuda_device):
    """Rows share blocks, reductions and 16-byte packs with their neighbours, but no values."""
    from cases.layernorm import native
    x, w, b, dy = inputs(rows, D, torch.bfloat16, torch.bfloat16, 11)
    y, stats = native.ln_forward(x, w, b, EPS)
    dx = native.ln_backward(dy, x, w, stats, (True, False, False))[0]
    bad = [1, 6, rows // 2, rows - 1]
    x[bad, 0], x[bad, D - 1] = float("nan"), float("inf")
    yb, sb = native.ln_forward(x, w, b, EPS)
    dxb = native.ln_backward(dy, x, w, sb, (True, False, False))[0]
    fine = torch.ones(rows, dtype=torch.bool, device="cuda")
    fine[bad] = False
    assert torch.isnan(yb[bad]).all() and torch.isnan(dxb[bad]).all()
    assert torch.equal(yb[fine], y[fine]) and torch.equal(dxb[fine], dx[fine])
