"""Token log-probabilities and the two losses on the GPU against 64-bit implementations."""
import math

import pytest
import torch

from lm_util import DTYPES, U32, assert_within, rounded

pytestmark = pytest.mark.gpu

IGNORE = -100


def inputs(B, T, V, dtype, seed, scored=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    labels = torch.randint(0, V, (B, T), device="cuda", generator=g)
    x = 2 * torch.randn(B, T, V, device="cuda", generator=g)
    x.scatter_add_(2, labels[..., None], 6 + 2 * torch.randn(B, T, 1, device="cuda", generator=g))
    keep = torch.rand(B, T, device="cuda", generator=g) < scored
    return x.to(dtype), torch.where(keep, labels, IGNORE), g


def logprob64(x, labels):
    """log softmax(x)[label] in fp64, differentiable; 0 where not scored."""
    ls = torch.log_softmax(x, dim=-1)
    lp = ls.gather(-1, labels.clamp(min=0)[..., None])[..., 0]
    return torch.where(labels != IGNORE, lp, torch.zeros_like(lp))


def lp_error(x, labels):
    """Bound of the kernel's log-probability error.  Every exp(x - m) carries the rounding of its
    exponent, at most U32 |x - m| log2(e) ln 2 relative, and 2^-22 of the approximation, so the
    sum's terms carry at most (spread + 8) U32 of themselves; partial sums add at most V / 256 + 64
    roundings of positive terms; log and the subtractions round values of at most |x_l - m| +
    log V."""
    x = x.double()
    m = x.amax(-1)
    V = x.size(-1)
    fin = torch.where(torch.isfinite(x), x, m[..., None])
    # Terms weighed by their share: sum p |x - m| is at most log V + 1 + ... <= 40 here.
    p = torch.softmax(fin, -1)
    spread = (p * (fin - m[..., None]).abs()).sum(-1)
    lead = x.gather(-1, labels.clamp(min=0)[..., None])[..., 0] - m
    lead = torch.where(torch.isfinite(lead), lead, torch.zeros_like(lead))
    return U32 * (2 * spread + V / 256 + 80 + 2 * (lead.abs() + math.log(V) + 1))


def grad_bound(want, p, c, spread, dtype, V):
    """c p: the exponent's rounding (|x - m| <= spread), the approximation, 1 / s and products; and
    at the label c - c p.  Then one rounding."""
    return U32 * (2 * spread + V / 256 + 100) * c.abs() * p \
        + 2 * U32 * want.abs() + rounded(want, dtype)


SHAPES = [(1, 1, 1), (1, 1, 2), (2, 3, 5), (1, 7, 100), (4, 1, 1023), (2, 2, 4096), (3, 5, 4097),
          (1, 2, 8191), (2, 1, 50001), (1, 1, 131071), (1, 3, 131072), (8, 40, 1000),
          (2, 300, 257)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,V", SHAPES)
def test_logprob_and_gradient(B, T, V, dtype, cuda_device):
    from cases.token_logprob.op import token_logprob
    x, labels, g = inputs(B, T, V, dtype, B * 100 + T + V)
    up = torch.randn(B, T, device="cuda", generator=g)
    x64 = x.double().requires_grad_(True)
    want = logprob64(x64, labels)
    want.backward(up.double())
    leaf = x.clone().requires_grad_(True)
    lp = token_logprob(leaf, labels, IGNORE)
    lp.backward(up)
    assert lp.dtype == torch.float32 and leaf.grad.dtype == dtype
    assert_within("logprob", lp, want, lp_error(x, labels) + rounded(want, torch.float32))
    p = torch.softmax(x.double(), -1)
    spread = (x.double().amax(-1, keepdim=True) - x.double())
    c = torch.where(labels != IGNORE, up.double(), 0.0)[..., None]
    assert_within("dlogits", leaf.grad, x64.grad,
                  grad_bound(x64.grad, p, c, spread, dtype, V) + 3 * U32 * c.abs() * (x64.grad != 0))
    assert not leaf.grad[labels == IGNORE].any()
    with torch.no_grad():
        assert torch.equal(token_logprob(leaf, labels, IGNORE), lp.detach())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,V", [(9, 250, 517), (2, 1000, 33), (5, 420, 9001)])
def test_many_rows(B, T, V, dtype, cuda_device):
    """Rows for every CTA that the SMs hold, and for several of each."""
    test_logprob_and_gradient(B, T, V, dtype, cuda_device)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_and_extreme_logits(dtype, cuda_device):
    """-inf and the type's lowest value in masked places, a leading label, infinities and NaN."""
    from cases.token_logprob.op import token_logprob
    low = torch.finfo(dtype).min
    V = 600
    x = torch.zeros(9, V, dtype=dtype, device="cuda")
    labels = torch.arange(9, device="cuda") * 50
    x[0, 100:] = -math.inf        # part of the vocabulary masked
    x[1, 100:] = low
    x[2] = -math.inf              # only the label is left
    x[2, 100] = 1.5
    x[3] = -math.inf              # nothing is left: NaN
    x[4, 200] = 80.0              # label leads by far
    x[5, 250] = -math.inf         # the label itself is masked
    x[6, 3] = math.inf            # NaN
    x[7, 9] = math.nan
    x[8] = low                    # all at the lowest value: uniform
    labels[0] = 5
    labels[1] = 7
    want = torch.log_softmax(x.double(), -1).gather(1, labels[:, None])[:, 0]
    leaf = x.clone().requires_grad_(True)
    lp = token_logprob(leaf, labels, IGNORE)
    lp.backward(torch.ones_like(lp))
    assert_within("logprob", lp, want, 200 * U32 * (1 + want.abs().nan_to_num(0, 0, 0)))
    lp = lp.detach()
    assert float(lp[2]) == 0.0 and float(lp[5]) == -math.inf
    assert torch.isnan(lp[[3, 6, 7]]).all()
    for r in (0, 1, 2, 4, 8):
        assert torch.isfinite(leaf.grad[r]).all()
    assert not leaf.grad[0, 100:].any() and not leaf.grad[1, 100:].any()


def test_label_out_of_range_is_nan(cuda_device):
    from cases.token_logprob.op import token_logprob
    x, labels, _ = inputs(1, 6, 300, torch.bfloat16, 1, scored=2.0)
    labels[0, 2], labels[0, 4] = 300, -7
    leaf = x.requires_grad_(True)
    lp = token_logprob(leaf, labels, IGNORE)
    assert torch.isnan(lp[0, [2, 4]]).all() and torch.isfinite(lp[0, [0, 1, 3, 5]]).all()
    lp.sum().backward()
    assert torch.isfinite(leaf.grad).all()


def test_other_ignore_index_may_be_a_token(cuda_device):
    from cases.token_logprob.op import token_logprob
    x, labels, _ = inputs(1, 40, 30, torch.float32, 2, scored=2.0)
    labels[0, ::3] = 0
    lp = token_logprob(x, labels, 0)
    assert not lp[labels == 0].any() and (lp[labels != 0] < 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_logits(dtype, cuda_device):
    """Views that shift positions, skip rows, cut the vocabulary or start off alignment."""
    from cases.token_logprob.op import token_logprob
    x, labels, _ = inputs(4, 10, 1030, dtype, 3)
    labels = labels % 900
    views = [(x[:, :-1], labels[:, 1:]), (x[:, 1:, :901], labels[:, 1:]),
             (x[:, ::2, 3:1003], labels[:, ::2]), (x.transpose(0, 1), labels.t()),
             (x[1], labels[1]), (x.view(2, 2, 10, 1030), labels.reshape(2, 2, 10)),
             (x[0:1].expand(4, 10, 1030), labels), (x.permute(0, 2, 1)[:, :, :5].permute(0, 2, 1), labels[:, :5])]
    for v, lab in views:
        lab = torch.where(lab < 0, IGNORE, lab)
        leaf = v.detach().requires_grad_(True)
        lp = token_logprob(leaf, lab, IGNORE)
        flat = v.contiguous().detach().requires_grad_(True)
        ref = token_logprob(flat, lab.contiguous(), IGNORE)
        assert_within("logprob", lp, ref, 64 * U32 * (1 + ref.abs()))
        lp.sum().backward()
        ref.sum().backward()
        assert_within("dlogits", leaf.grad, flat.grad,
                      64 * U32 * flat.grad.double().abs() + 2 * rounded(flat.grad, dtype))


def preference64(lp, ref, labels, beta, s):
    d = torch.where(labels != IGNORE, lp - ref.double(), 0.0)
    r = beta * d.sum(1)
    P = r.numel() // 2
    z = r[:P] - r[P:]
    ls = torch.nn.functional.logsigmoid
    return (-(1 - s) * ls(z) - s * ls(-z)).mean(), r


def policy64(lp, old, ref, adv, labels, lo, hi, k):
    m = labels != IGNORE
    n = m.sum().clamp(min=1)
    a = adv.double() if adv.dim() == 2 else adv.double()[:, None]
    ratio = torch.exp(torch.where(m, lp - old.double(), 0.0))
    d = torch.where(m, ref.double() - lp, 0.0)
    kl = torch.expm1(d) - d
    gain = torch.minimum(ratio * a, ratio.clamp(1 - lo, 1 + hi) * a)
    return torch.where(m, k * kl - gain, 0.0).sum() / n, (kl * m).sum() / n


LOSS_SHAPES = [(2, 1, 50), (4, 33, 1001), (6, 40, 512), (2, 600, 130), (300, 3, 64), (16, 64, 2048)]


def check_logits_gradient(leaf, x64, lp64, coef64, extra, dtype):
    """The gradient's bound: token_logprob's for the exact coefficient, plus the coefficient's own
    error ``extra`` times |onehot - softmax|."""
    V = leaf.size(-1)
    p = torch.softmax(x64.detach(), -1)
    spread = x64.detach().amax(-1, keepdim=True) - x64.detach()
    c = coef64[..., None]
    unit = torch.where(c != 0, x64.grad / c, p).abs()
    bound = grad_bound(x64.grad, p, c, spread, dtype, V) + 3 * U32 * c.abs() * (x64.grad != 0)
    assert_within("dlogits", leaf.grad, x64.grad, bound + extra[..., None] * unit)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,V", LOSS_SHAPES)
def test_preference_loss(B, T, V, dtype, cuda_device):
    from cases.preference_loss.op import preference_loss
    x, labels, g = inputs(B, T, V, dtype, B + T + V)
    labels[0] = IGNORE  # an answer without any scored position
    beta, s = 0.25, 0.1
    with torch.no_grad():
        ref = (logprob64(x.double(), labels) + 0.3 * torch.randn(B, T, device="cuda", generator=g)).float()
    x64 = x.double().requires_grad_(True)
    lp64 = logprob64(x64, labels)
    lp64.retain_grad()
    want, reward64 = preference64(lp64, ref, labels, beta, s)
    (want * 3).backward()
    leaf = x.clone().requires_grad_(True)
    loss, reward = preference_loss(leaf, labels, ref, beta, s, IGNORE)
    assert not reward.requires_grad
    (loss * 3).backward()
    e = (lp_error(x, labels) * (labels != IGNORE)).sum(1) * beta  # of a reward
    e = e + 2 * U32 * reward64.abs()
    assert_within("reward", reward, reward64, e)
    P = B // 2
    ez = e[:P] + e[P:]
    assert_within("loss", loss, want, ez.mean() + 4 * U32 * want.abs())
    # d2 loss / dz2 <= 1/4
    extra = 3 * beta / P * (ez / 4).repeat(2)[:, None] + 4 * U32 * lp64.grad.abs()
    check_logits_gradient(leaf, x64, lp64, lp64.grad, extra * (labels != IGNORE), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per_token", [False, True])
@pytest.mark.parametrize("B,T,V", LOSS_SHAPES)
def test_policy_loss(B, T, V, per_token, dtype, cuda_device):
    from cases.policy_loss.op import policy_loss
    x, labels, g = inputs(B, T, V, dtype, B + T + V)
    labels[0] = IGNORE
    lo, hi, k = 0.2, 0.3, 0.1
    def rand(*sh):
        return torch.randn(*sh, device="cuda", generator=g)
    with torch.no_grad():
        lp = logprob64(x.double(), labels)
        move = 0.3 * rand(B, T).double()
        # At the border itself rounding decides the branch: keep 1e-3 away.
        for border in (math.log(1 + hi), math.log(1 - lo)):
            move = torch.where((move - border).abs() < 1e-3, border + 2e-3, move)
        old, ref = (lp - move).float(), (lp + 0.4 * rand(B, T)).float()
        adv = rand(B, T) if per_token else rand(B)
    x64 = x.double().requires_grad_(True)
    lp64 = logprob64(x64, labels)
    lp64.retain_grad()
    want, kl64 = policy64(lp64, old, ref, adv, labels, lo, hi, k)
    (want * 2).backward()
    leaf = x.clone().requires_grad_(True)
    loss, kl = policy_loss(leaf, labels, old, ref, adv, lo, hi, k, IGNORE)
    assert not kl.requires_grad
    (loss * 2).backward()
    m = labels != IGNORE
    n = m.sum().clamp(min=1)
    e = lp_error(x, labels) * m
    a = (adv if per_token else adv[:, None]).double().abs()
    # ratio <= e^1.5 and e^d <= e^2 at these spreads; their slopes in lp are themselves.
    assert_within("kl", kl, kl64, (e * 8).sum() / n + 4 * U32 * kl64.abs())
    assert_within("loss", loss, want, (e * (8 * k + 5 * a)).sum() / n + 4 * U32 * want.abs()
                  + 4 * U32 * (5 * a * m).sum() / n)
    extra = 2 * e * (8 * k + 5 * a) / n + 6 * U32 * (2 * m * (8 * k + 5 * a) / n)
    check_logits_gradient(leaf, x64, lp64, lp64.grad, extra, dtype)


def test_logprob_past_fp32(cuda_device):
    """A log-probability that overflows fp32 is -inf, and so is its answer's reward (not NaN)."""
    from cases.preference_loss.op import preference_loss
    from cases.token_logprob.op import token_logprob
    x = torch.zeros(2, 1, 4, device="cuda")
    x[0, 0, 0], x[0, 0, 1] = -3.4e38, 3e38
    labels = torch.zeros(2, 1, dtype=torch.long, device="cuda")
    assert float(token_logprob(x, labels)[0]) == -math.inf
    loss, reward = preference_loss(x, labels, torch.zeros(2, 1, device="cuda"))
    assert float(reward[0]) == -math.inf and float(loss) == math.inf
    assert abs(float(reward[1]) + 0.1 * math.log(4)) < 1e-7


def test_nothing_scored(cuda_device):
    from cases.policy_loss.op import policy_loss
    from cases.preference_loss.op import preference_loss
    x = torch.randn(2, 5, 40, device="cuda", requires_grad=True)
    labels = torch.full((2, 5), IGNORE, device="cuda")
    zero = torch.zeros(2, 5, device="cuda")
    loss, reward = preference_loss(x, labels, zero)
    assert abs(float(loss) - math.log(2)) < 1e-6 and not reward.any()
    loss.backward()
    assert not x.grad.any()
    x.grad = None
    loss, kl = policy_loss(x, labels, zero, zero, torch.ones(2, device="cuda"))
    assert float(loss) == 0.0 and float(kl) == 0.0
    loss.backward()
    assert not x.grad.any()


def test_extreme_rewards(cuda_device):
    """z far beyond exp's range either way: the loss is linear or 0, its gradient finite."""
    from cases.preference_loss.op import preference_loss
    x = torch.randn(4, 3, 50, device="cuda")
    labels = torch.randint(0, 50, (4, 3), device="cuda")
    ref = torch.zeros(4, 3, device="cuda")
    ref[0], ref[1] = 1e5, -1e5
    leaf = x.clone().requires_grad_(True)
    loss, reward = preference_loss(leaf, labels, ref, 1.0)
    want, r64 = preference64(logprob64(x.double(), labels), ref, labels, 1.0, 0.0)
    assert_within("loss", loss, want, 1e-6 * want.abs())
    loss.backward()
    assert torch.isfinite(leaf.grad).all() and not leaf.grad[1].any() and leaf.grad[0].any()


def test_loss_needs_no_gradient(cuda_device):
    from cases.policy_loss.op import policy_loss
    from cases.preference_loss.op import preference_loss
    x, labels, _ = inputs(2, 4, 100, torch.float32, 1)
    z = torch.zeros(2, 4, device="cuda")
    assert not preference_loss(x, labels, z)[0].requires_grad
    assert not policy_loss(x, labels, z, z, z)[0].requires_grad


@pytest.mark.parametrize("which", ["logprob", "preference", "policy"])
def test_captured_and_replayed_on_new_data(which, cuda_device):
    from cases.policy_loss import native as pol
    from cases.preference_loss import native as pref
    from cases.token_logprob import native as lp
    x, labels, g = inputs(4, 60, 3001, torch.bfloat16, 8)
    ref, old, adv = (0.1 * torch.randn(4, 60, device="cuda", generator=g) - 3 for _ in range(3))
    sx, sl = torch.zeros_like(x), torch.zeros_like(labels)

    def step(x, labels):
        if which == "logprob":
            out, stats = lp.logprob_forward(x, labels, IGNORE)
            return out, lp.logprob_backward(x, labels, stats, ref, IGNORE)
        if which == "preference":
            loss, r, state = pref.preference_forward(x, labels, ref, 0.1, 0.0, IGNORE)
            return loss, r, pref.preference_backward(x, labels, state, None, IGNORE)
        loss, kl, state = pol.policy_forward(x, labels, old, ref, adv, 0.2, 0.2, 0.1, IGNORE)
        return loss, kl, pol.policy_backward(x, labels, state, None, IGNORE)

    want = step(x, labels)
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(sx, sl)
        graphs.append((graph, out))
    sx.copy_(x)
    sl.copy_(labels)
    for graph, out in graphs * 2:
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("name", ["token_logprob", "preference_loss", "policy_loss"])
def test_verify_all_passes(name, cuda_device):
    import importlib
    from framework.verify import verify_all
    case = importlib.import_module(f"cases.{name}").CASE
    op = importlib.import_module(f"cases.{name}.op")
    ok, report = verify_all(case, op.candidate, device="cuda")
    assert ok, report


@pytest.mark.parametrize("dtype", DTYPES)
def test_unscored_positions_are_not_read(dtype, cuda_device):
    """NaN and infinities in the logits, scores and advantages of unscored positions change nothing."""
    from cases.policy_loss.op import policy_loss
    from cases.preference_loss.op import preference_loss
    x, labels, g = inputs(4, 9, 700, dtype, 6)
    scored = labels != IGNORE
    ref, old, adv = (torch.randn(4, 9, device="cuda", generator=g) for _ in range(3))

    def run(x, ref, old, adv):
        leaf = x.clone().requires_grad_(True)
        a = preference_loss(leaf, labels, ref)
        b = policy_loss(leaf, labels, old, ref, adv, kl_coef=0.1)
        (a[0] + b[0]).backward()
        return a[0], a[1], b[0], b[1], leaf.grad

    want = run(x, ref, old, adv)
    bad = x.clone()
    bad[~scored] = math.nan
    spoil = [torch.where(scored, t, v) for t, v in ((ref, math.nan), (old, math.inf), (adv, math.nan))]
    for p, q in zip(want, run(bad, *spoil)):
        assert torch.equal(p, q)


def test_empty_batches(cuda_device):
    from cases.policy_loss.op import policy_loss
    from cases.preference_loss.op import preference_loss
    from cases.token_logprob.op import token_logprob
    for B, T in ((2, 0), (0, 5)):
        x = torch.randn(B, T, 30, device="cuda", requires_grad=True)
        lab = torch.zeros(B, T, dtype=torch.int64, device="cuda")
        z = torch.zeros(B, T, device="cuda")
        assert token_logprob(x, lab).shape == (B, T)
        loss, reward = preference_loss(x, lab, z)
        assert reward.shape == (B,)
        assert (abs(float(loss.detach()) - math.log(2)) < 1e-6) if B else torch.isnan(loss)
        loss.backward()
        assert x.grad.shape == x.shape
        loss, kl = policy_loss(x, lab, z, z, torch.ones(B, device="cuda"))
        assert float(loss.detach()) == 0.0 and float(kl) == 0.0


def test_offsets_past_32_bits(cuda_device):
    """A view whose rows lie 2^31 elements and more behind its start."""
    from cases.token_logprob import native
    V = 70000
    rows = (1 << 31) // V + 40
    base = torch.zeros(rows, V, dtype=torch.bfloat16, device="cuda")
    x, labels, g = inputs(1, 30, V, torch.bfloat16, 2, scored=0.8)
    base[-30:] = x[0]
    lab = torch.full((rows,), IGNORE, device="cuda")
    lab[-30:] = labels[0]
    lab[0] = 17
    lp, stats = native.logprob_forward(base, lab, IGNORE)
    small, sstats = native.logprob_forward(x[0], labels[0], IGNORE)
    assert_within("logprob", lp[-30:], small, 200 * U32 * (1 + small.abs()))
    assert abs(float(lp[0]) + math.log(V)) < 1e-5
    up = torch.ones_like(lp)
    dx = native.logprob_backward(base, lab, stats, up, IGNORE)
    want = native.logprob_backward(x[0], labels[0], sstats, up[-30:], IGNORE)
    # Equal up to the sums' grouping: two roundings to bf16 apart at most.
    assert_within("dlogits", dx[-30:], want, 2.01 * rounded(want, torch.bfloat16) + 1e-9)
    assert not dx[1:-30].any() and dx[0].any()


def test_other_streams(cuda_device):
    from cases.policy_loss.op import policy_loss
    x, labels, g = inputs(4, 50, 2001, torch.bfloat16, 4)
    z = torch.full((4, 50), -3.0, device="cuda")
    adv = torch.randn(4, device="cuda", generator=g)

    def run():
        leaf = x.clone().requires_grad_(True)
        loss, kl = policy_loss(leaf, labels, z, z, adv, kl_coef=0.1)
        loss.backward()
        return loss.detach(), kl, leaf.grad

    want = run()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(run())
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want))


def test_state_of_another_device_is_refused(cuda_device):
    """The backwards without autograd take the forward's state; its address has to be the GPU's."""
    from cases.policy_loss import native as policy
    from cases.preference_loss import native as preference
    from cases.token_logprob import native as logprob
    x = torch.randn(2, 3, 40, device="cuda")
    labels, zero = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(2, 3, device="cuda")
    state = preference.preference_forward(x, labels, zero, 0.1, 0.0, -100)[2]
    with pytest.raises(RuntimeError, match="state must be a CUDA tensor"):
        preference.preference_backward(x, labels, state.cpu(), None, -100)
    state = policy.policy_forward(x, labels, zero, zero, torch.ones(2, device="cuda"), 0.2, 0.2, 0.0, -100)[2]
    with pytest.raises(RuntimeError, match="state must be a CUDA tensor"):
        policy.policy_backward(x, labels, state.cpu(), None, -100)
    stats = logprob.logprob_forward(x, labels, -100)[1]
    with pytest.raises(RuntimeError, match="stats must be a CUDA tensor"):
        logprob.logprob_backward(x, labels, stats.cpu(), zero, -100)
