"""Cases of the language-model operators: layer norm, the log-probabilities of chosen tokens, the
preference loss, the clipped policy loss and the Newton-Schulz orthogonalisation of an update.

``listed()`` and ``draw(rng)`` give cases, ``prepare(case, seed)`` makes a case's inputs on the
GPU, and ``run(state)`` takes one pass through the operator: in its plain form (elementary torch
operations in fp32, rounded once at the end) or, with ``own`` set, through the package's public
calls.  ``work(case)`` is the traffic and arithmetic that a pass cannot do without, and
``exact(case, seed)`` the outputs from the definitions in 64 bits.
"""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
IGNORE = -100  # the label of a position that is not scored (prompt, padding)
LN_EPS = 1e-5
BETA, SMOOTHING = 0.1, 0.05  # preference loss: reward scale, label smoothing
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04  # policy loss
NS_STEPS, NS_EPS = 5, 1e-7
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


# ---------------------------------------------------------------------------------- the cases

def listed():
    return [
        # Serving: one token of each of 8 sequences through a normalisation (latency).
        {"name": "layernorm_tokens", "op": "layernorm", "rows": 8, "d": 4096,
         "dtype": "bfloat16", "train": False},
        # Training: one normalisation of a block over 8192 tokens, with every gradient.
        {"name": "layernorm_train", "op": "layernorm", "rows": 8192, "d": 4096,
         "dtype": "bfloat16", "train": True},
        # A full-precision normalisation whose rows share no alignment.
        {"name": "layernorm_ragged", "op": "layernorm", "rows": 4099, "d": 1023,
         "dtype": "float32", "train": True},
        # Scoring one answer token of 4 prompts over a large vocabulary (few, long rows).
        {"name": "logprob_answers", "op": "logprob", "batch": 4, "t": 1, "vocab": 131071,
         "dtype": "float32", "train": True},
        # The reference model's pass of a preference run: scores only, no gradient.
        {"name": "logprob_reference", "op": "logprob", "batch": 16, "t": 512, "vocab": 32768,
         "dtype": "bfloat16", "train": False},
        # A debugging-size preference step (2 pairs, short answers).
        {"name": "preference_short", "op": "preference", "batch": 4, "t": 33, "vocab": 8191,
         "dtype": "float16", "train": True},
        # A preference step of 8 pairs.
        {"name": "preference_train", "op": "preference", "batch": 16, "t": 1024, "vocab": 32768,
         "dtype": "bfloat16", "train": True},
        # A policy step from full-precision logits with an odd vocabulary.
        {"name": "policy_odd", "op": "policy", "batch": 8, "t": 250, "vocab": 50001,
         "dtype": "float32", "train": True},
        # A policy step of 16 long answers over a large vocabulary: the largest loss.
        {"name": "policy_train", "op": "policy", "batch": 16, "t": 1024, "vocab": 131072,
         "dtype": "bfloat16", "train": True},
        # The update of four small projections at once (latency).
        {"name": "orthogonalize_small", "op": "orthogonalize", "batch": 4, "m": 256, "n": 256,
         "dtype": "bfloat16", "train": False},
        # A full-precision update whose sizes fill no tile.
        {"name": "orthogonalize_odd", "op": "orthogonalize", "batch": 1, "m": 2601, "n": 1001,
         "dtype": "float32", "train": False},
        # The update of a large projection.
        {"name": "orthogonalize_large", "op": "orthogonalize", "batch": 1, "m": 4096, "n": 8192,
         "dtype": "bfloat16", "train": False},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["layernorm", "logprob", "preference", "policy", "orthogonalize"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "layernorm":
        d = _log_uniform(rng, 48, 16384)
        rows = _log_uniform(rng, 1, min(32768, (1 << 26) // d))
        return {"op": op, "rows": rows, "d": d, "dtype": dtype, "train": rng.random() < 0.7}
    if op == "orthogonalize":
        m, n = _log_uniform(rng, 48, 4096), _log_uniform(rng, 48, 4096)
        batch = rng.randint(1, 6) if m * n <= 1 << 20 else 1
        return {"op": op, "batch": batch, "m": m, "n": n, "dtype": dtype, "train": False}
    vocab = _log_uniform(rng, 1000, 131072)
    batch = rng.randint(1, 16)
    if op == "preference":
        batch += batch % 2
    t = _log_uniform(rng, 1, max(1, min(1024, (1 << 28) // (vocab * batch))))
    train = op != "logprob" or rng.random() < 0.5
    return {"op": op, "batch": batch, "t": t, "vocab": vocab, "dtype": dtype, "train": train}


# --------------------------------------------------------------------------------- the inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _scores(logits, labels):
    """log softmax(logits)[label] by chunks of rows, 0 where the position is not scored."""
    flat, lab = logits.view(-1, logits.size(-1)), labels.view(-1)
    out = torch.zeros(lab.numel(), device=logits.device)
    step = max(1, (1 << 28) // flat.size(1))
    for i in range(0, flat.size(0), step):
        x = flat[i:i + step].float()
        at = lab[i:i + step].clamp(min=0)
        out[i:i + step] = x.gather(1, at[:, None])[:, 0] - x.logsumexp(1)
    return torch.where(lab != IGNORE, out, 0.0).view(labels.shape)


def _spans(case, gen):
    """[batch, t] truth values: each sequence's scored positions, after its prompt (up to a
    quarter) and before its padding (up to a quarter); three quarters on average."""
    b, t = case["batch"], case["t"]
    u = torch.rand(2, b, 1, device="cuda", generator=gen)
    at = torch.arange(t, device="cuda")[None]
    first, last = (u[0] * (t // 4 + 1)).floor(), t - (u[1] * (t // 4 + 1)).floor()
    return (at >= first) & (at < last)


def prepare(case, seed):
    g = _generator(seed)
    dtype, op = DTYPES[case["dtype"]], case["op"]
    randn = functools.partial(torch.randn, device="cuda", generator=g)
    if op == "layernorm":
        rows, d, train = case["rows"], case["d"], case["train"]
        # Activations: per-channel offsets and a few channels much larger than the others.
        scale = 1.0 + 9.0 * (torch.rand(d, device="cuda", generator=g) < 0.01)
        x = ((randn(rows, d) + 0.5 * randn(d)) * scale).to(dtype)
        w, b = (1.0 + 0.1 * randn(d)).to(dtype), (0.1 * randn(d)).to(dtype)
        dy = randn(rows, d).to(dtype)
        return {"op": op, "x": x.requires_grad_(train), "weight": w.requires_grad_(train),
                "bias": b.requires_grad_(train), "dy": dy, "train": train}
    if op == "orthogonalize":
        batch, m, n = case["batch"], case["m"], case["n"]
        # A momentum of gradients: some strong directions that fall off, and noise.
        k = min(m, n, 16)
        fall = 1.0 / torch.arange(1, k + 1, device="cuda")
        u = (randn(batch, m, k) * fall) @ randn(batch, k, n)
        update = (1e-3 * (u + 0.5 * randn(batch, m, n))).to(dtype)
        return {"op": op, "update": update[0] if batch == 1 else update}
    b, t, v = case["batch"], case["t"], case["vocab"]
    labels = torch.randint(0, v, (b, t), device="cuda", generator=g)
    logits = torch.empty(b, t, v, dtype=dtype, device="cuda")
    for i in range(b):
        logits[i] = 2.0 * randn(t, v)
    # The chosen token stands out, as in a trained model's scores.
    logits.scatter_add_(2, labels[..., None], (8.0 + 2.0 * randn(b, t, 1)).to(dtype))
    labels = torch.where(_spans(case, g), labels, IGNORE)
    state = {"op": op, "labels": labels, "train": case["train"]}
    scored = labels != IGNORE
    if op == "logprob":
        state["dlogprob"] = randn(b, t)
    elif op == "preference":
        state["ref"] = torch.where(scored, _scores(logits, labels) + 0.1 * randn(b, t), 0.0)
    else:
        s = _scores(logits, labels)
        move = 0.15 * randn(b, t)
        # On a clip border itself rounding would decide whether a token has a gradient.
        for border in (math.log(1 + CLIP_HIGH), math.log(1 - CLIP_LOW)):
            move = torch.where((move - border).abs() < 2e-3, border + 4e-3, move)
        state["old"] = torch.where(scored, s - move, 0.0)
        state["ref"] = torch.where(scored, s + 0.2 * randn(b, t), 0.0)
        state["advantage"] = randn(b)
    state["logits"] = logits.requires_grad_(case["train"])
    return state


# -------------------------------------------------------------------------------- the passes

@functools.cache
def _ops():
    """The package's public calls."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "nl2cuda-kernel-agent_b200"))
    from cases.layernorm.op import layer_norm
    from cases.orthogonalize.op import orthogonalize
    from cases.policy_loss.op import policy_loss
    from cases.preference_loss.op import preference_loss
    from cases.token_logprob.op import token_logprob
    return {"layernorm": layer_norm, "orthogonalize": orthogonalize, "policy": policy_loss,
            "preference": preference_loss, "logprob": token_logprob}


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    f = _ops()[s["op"]]
    if s["op"] == "layernorm":
        if not s["train"]:
            with torch.no_grad():
                return {"y": f(s["x"], s["weight"], s["bias"], LN_EPS)}
        y = f(s["x"], s["weight"], s["bias"], LN_EPS)
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    if s["op"] == "orthogonalize":
        return {"out": f(s["update"], steps=NS_STEPS, coefficients=NS_COEFFICIENTS, eps=NS_EPS)}
    if s["op"] == "logprob":
        if not s["train"]:
            with torch.no_grad():
                return {"logprob": f(s["logits"], s["labels"], ignore_index=IGNORE)}
        lp = f(s["logits"], s["labels"], ignore_index=IGNORE)
        (dx,) = torch.autograd.grad(lp, (s["logits"],), s["dlogprob"])
        return {"logprob": lp.detach(), "dlogits": dx}
    if s["op"] == "preference":
        loss, reward = f(s["logits"], s["labels"], s["ref"], beta=BETA,
                         label_smoothing=SMOOTHING, ignore_index=IGNORE)
        (dx,) = torch.autograd.grad(loss, (s["logits"],))
        return {"loss": loss.detach(), "reward": reward, "dlogits": dx}
    loss, kl = f(s["logits"], s["labels"], s["old"], s["ref"], s["advantage"],
                 clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF, ignore_index=IGNORE)
    (dx,) = torch.autograd.grad(loss, (s["logits"],))
    return {"loss": loss.detach(), "kl": kl, "dlogits": dx}


@torch.no_grad()
def _run_plain(s):
    return {"layernorm": _plain_layernorm, "orthogonalize": _plain_orthogonalize,
            "logprob": _plain_logprob, "preference": _plain_preference,
            "policy": _plain_policy}[s["op"]](s)


def _plain_layernorm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    dtype = s["x"].dtype
    c = x - x.mean(1, keepdim=True)
    rstd = (c.square().mean(1, keepdim=True) + LN_EPS).rsqrt()
    xh = c * rstd
    y = (xh * w + b).to(dtype)
    if not s["train"]:
        return {"y": y}
    dy = s["dy"].float()
    gw = dy * w
    dx = (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True)) * rstd
    return {"y": y, "dx": dx.to(dtype), "dw": (dy * xh).sum(0).to(dtype),
            "db": dy.sum(0).to(dtype)}


def _softmax_parts(s):
    """exp(logits - their maximum) and its sum, each position's label (0 where it is not scored),
    whether it is scored, and its log-probability."""
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    x = x - m
    scored = s["labels"] != IGNORE
    at = torch.where(scored, s["labels"], 0)[..., None]
    chosen = x.gather(-1, at)[..., 0]
    p = x.exp_()
    total = p.sum(-1, keepdim=True)
    lp = torch.where(scored, chosen - total[..., 0].log(), 0.0)
    return p, total, at, scored, lp


def _logit_gradient(p, total, at, coefficient, dtype):
    """coefficient * (one-hot of the label - softmax)."""
    c = coefficient[..., None]
    return p.mul_(-c / total).scatter_add_(-1, at, c).to(dtype)


def _plain_logprob(s):
    p, total, at, scored, lp = _softmax_parts(s)
    if not s["train"]:
        return {"logprob": lp}
    c = torch.where(scored, s["dlogprob"], 0.0)
    return {"logprob": lp, "dlogits": _logit_gradient(p, total, at, c, s["logits"].dtype)}


def _plain_preference(s):
    p, total, at, scored, lp = _softmax_parts(s)
    # Sums over long answers, whose differences are small, in 64 bits.
    reward = BETA * torch.where(scored, lp.double() - s["ref"].double(), 0.0).sum(1)
    pairs = reward.numel() // 2
    z = reward[:pairs] - reward[pairs:]
    up, down = torch.sigmoid(-z), torch.sigmoid(z)  # -d/dz log sigmoid(z), d/dz of the other
    softplus = lambda v: v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731
    loss = ((1 - SMOOTHING) * softplus(-z) + SMOOTHING * softplus(z)).mean()
    dz = (SMOOTHING * down - (1 - SMOOTHING) * up) / pairs
    c = torch.cat((dz, -dz))[:, None] * BETA * scored
    return {"loss": loss.float(), "reward": reward.float(),
            "dlogits": _logit_gradient(p, total, at, c.float(), s["logits"].dtype)}


def _plain_policy(s):
    p, total, at, scored, lp = _softmax_parts(s)
    a = s["advantage"][:, None].double()
    lp64, count = lp.double(), scored.sum().clamp(min=1)
    ratio = (lp64 - s["old"].double()).exp()
    clipped = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    behind = s["ref"].double() - lp64
    kl = behind.exp() - behind - 1
    gain = torch.minimum(ratio * a, clipped * a)
    mean = lambda v: (torch.where(scored, v, 0.0).sum() / count).float()  # noqa: E731
    free = ratio * a <= clipped * a  # the unclipped term decides
    c = (torch.where(free, -ratio * a, 0.0) + KL_COEF * (1 - behind.exp())) / count
    c = torch.where(scored, c, 0.0).float()
    return {"loss": mean(KL_COEF * kl - gain), "kl": mean(kl),
            "dlogits": _logit_gradient(p, total, at, c, s["logits"].dtype)}


def _ns_step(x, coefficients):
    a, b, c = coefficients
    g = x @ x.mT
    return a * x + (b * g + c * (g @ g)) @ x


def _plain_orthogonalize(s):
    x = s["update"].float()
    tall = x.size(-2) > x.size(-1)
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS)
    x = functools.reduce(_ns_step, [NS_COEFFICIENTS] * NS_STEPS, x)
    return {"out": (x.mT if tall else x).to(s["update"].dtype).contiguous()}


# ----------------------------------------------------------------------- work and definitions

def work(case):
    e = DTYPES[case["dtype"]].itemsize
    if case["op"] == "layernorm":
        n, d = case["rows"] * case["d"], case["d"]
        # Forward: x, y.  Backward: x, dy, dx.
        return {"bytes": e * (n * (5 if case["train"] else 2) + 4 * d),
                "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "orthogonalize":
        m, n = sorted((case["m"], case["n"]))
        # Per step: X X^T and its square (symmetric: half of each), and the product with X.
        return {"bytes": 2 * e * case["batch"] * m * n,
                "flops": NS_STEPS * case["batch"] * (3 * m * m * n + m ** 3)}
    b, t, v = case["batch"], case["t"], case["vocab"]
    rows = b * t
    scored = max(1, round(0.75 * rows))
    # Scored rows are read by each pass; a gradient is written for every row.
    reads, writes = (2, 1) if case["train"] else (1, 0)
    return {"bytes": e * v * (reads * scored + writes * rows) + 20 * rows,
            "flops": v * scored * (8 if case["train"] else 4)}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    return {"layernorm": _exact_layernorm, "orthogonalize": _exact_orthogonalize}.get(
        s["op"], _exact_loss)(s)


def _exact_layernorm(s):
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    sd = torch.sqrt(var + LN_EPS)
    y = (x - mean) / sd * w + b
    if not s["train"]:
        return {"y": y}
    dy = s["dy"].double()
    d, h = x.size(1), (x - mean) / sd
    t = dy * w
    dx = (d * t - t.sum(1, keepdim=True) - h * (t * h).sum(1, keepdim=True)) / (d * sd)
    return {"y": y, "dx": dx, "dw": torch.einsum("nd,nd->d", dy, h), "db": dy.sum(0)}


def _exact_orthogonalize(s):
    g = s["update"].double()
    x = g / (torch.linalg.matrix_norm(g, keepdim=True) + NS_EPS)
    a, b, c = NS_COEFFICIENTS
    eye = torch.eye(min(g.shape[-2:]), dtype=torch.float64, device=g.device)
    for _ in range(NS_STEPS):
        if x.size(-2) <= x.size(-1):
            k = torch.matmul(x, x.transpose(-1, -2))
            x = torch.matmul(a * eye + torch.matmul(k, b * eye + c * k), x)
        else:
            k = torch.matmul(x.transpose(-1, -2), x)
            x = torch.matmul(x, a * eye + torch.matmul(k, b * eye + c * k))
    return {"out": x}


def _exact_loss(s):
    logits, labels = s["logits"].detach(), s["labels"]
    b, t, v = logits.shape
    flat, lab = logits.view(-1, v), labels.view(-1)
    scored = lab.ne(IGNORE)
    lp = torch.zeros(b * t, dtype=torch.float64, device=logits.device)
    step = max(1, (1 << 27) // v)
    for i in range(0, b * t, step):
        ls = torch.log_softmax(flat[i:i + step].double(), 1)
        lp[i:i + step] = ls.gather(1, lab[i:i + step].clamp(min=0)[:, None])[:, 0]
    lp = (lp * scored).view(b, t).requires_grad_(True)
    mask = scored.view(b, t).double()
    with torch.enable_grad():
        if s["op"] == "logprob":
            out = {"logprob": lp}
            target = (lp * s["dlogprob"].double() * mask).sum()
        elif s["op"] == "preference":
            r = BETA * ((lp - s["ref"].double()) * mask).sum(1)
            win, lose = r.chunk(2)
            ls = torch.nn.functional.logsigmoid
            target = -((1 - SMOOTHING) * ls(win - lose) + SMOOTHING * ls(lose - win)).mean()
            out = {"loss": target, "reward": r}
        else:
            n = mask.sum().clamp(min=1)
            a = s["advantage"].double()[:, None]
            ratio = torch.exp(lp - s["old"].double())
            gain = torch.minimum(ratio * a, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a)
            d = s["ref"].double() - lp
            kl = (mask * (torch.expm1(d) - d)).sum() / n
            target = KL_COEF * kl - (mask * gain).sum() / n
            out = {"loss": target, "kl": kl}
        (c,) = torch.autograd.grad(target, (lp,))
    out = {k: x.detach() for k, x in out.items()}
    if not s["train"]:
        return out
    c = (c * mask).view(-1, 1)
    dx = torch.empty(b * t, v, dtype=torch.float64, device=logits.device)
    for i in range(0, b * t, step):
        p = torch.softmax(flat[i:i + step].double(), 1)
        p.scatter_add_(1, lab[i:i + step].clamp(min=0)[:, None],
                       torch.full_like(p[:, :1], -1.0))
        dx[i:i + step] = p * -c[i:i + step]
    out["dlogits"] = dx.view(b, t, v)
    return out
