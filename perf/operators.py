"""Cases of the read encoder's operators: the linear layer, the layer norm and the softmax loss.

The index is built over vectors that a signal encoder makes of reads: windows of 2,000 samples
become 400 tokens each, a convolutional front end is projected to 256 features, and pre-norm
blocks (layer norm, 256 -> 1,024 -> 256 feed-forward with GELU, residual sums) end in a mean over
the window.  The encoder learns by telling each window's partner from every other vector of a
bank, a softmax over as many classes as the bank has rows.  The three operators here are the ones
that path spends its products and its bytes on, forward for encoding and with their gradients for
training:

  linear        y = act(x w^T + b) + residual                      torch.ops.rbq.linear
  layer_norm    y = (x - mean) rstd * w + b                        torch.ops.rbq.layer_norm
  softmax_loss  loss_i = logsumexp_j(scale q_i.k_j) - scale q_i.k_t(i)   torch.ops.rbq.softmax_loss

`run` computes them from elementary torch operations in 32 bits, or, where `own` is true, through
the framework's operators.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
EPS = 1e-5
SCALE = 1.0 / 0.07  # the usual temperature of a contrastive loss


def _linear(name, m, k, n, dtype, act, residual, train):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "residual": residual,
            "train": train}


def _norm(name, rows, d, dtype, train):
    return {"name": name, "op": "layer_norm", "rows": rows, "d": d, "dtype": dtype, "train": train}


def _loss(name, n, v, d, dtype, train):
    return {"name": name, "op": "softmax_loss", "n": n, "v": v, "d": d, "dtype": dtype, "train": train}


def listed():
    return [
        # the feed-forward's first layer on one window (400 tokens): a single read encoded as it arrives
        _linear("linear one window", 400, 256, 1024, "fp16", "gelu", False, False),
        # the same layer on an encoding batch of 2,048 windows
        _linear("linear encode batch", 819200, 256, 1024, "fp16", "gelu", False, False),
        # the feed-forward's second layer with its residual sum, a training step on 128 windows
        _linear("linear down train", 51200, 1024, 256, "bf16", "none", True, True),
        # the feed-forward's first layer, the same training step
        _linear("linear gelu train", 51200, 256, 1024, "fp16", "gelu", False, True),
        # sizes that no tile or vector divides: packed windows of ragged lengths, odd widths
        _linear("linear ragged train", 13331, 331, 517, "bf16", "relu", False, True),
        # one window's tokens before a block
        _norm("norm one window", 400, 256, "fp16", False),
        # an encoding batch of 2,048 windows
        _norm("norm encode batch", 819200, 256, "fp16", False),
        # a training step on 512 windows
        _norm("norm train", 204800, 256, "bf16", True),
        # an odd width in single precision
        _norm("norm ragged train", 5003, 771, "fp32", True),
        # validation of 64 windows against a small bank (1,024 rows, one per list of the 1M index)
        _loss("loss small bank", 64, 1024, 256, "fp16", False),
        # a training step against one row per list of the sharded index, at the reference's width
        _loss("loss lists train", 2048, 65536, 384, "bf16", True),
        # a training step against every read of the read-overlap workload
        _loss("loss reads train", 8192, 200000, 256, "fp16", True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["linear", "layer_norm", "softmax_loss"])
    train = rng.random() < 0.6
    if op == "linear":
        k, n = _log_int(rng, 1, 1280), _log_int(rng, 1, 1280)
        if rng.random() < 0.5:  # widths are mostly whole vectors, as a model's are
            k, n = -(-k // 8) * 8, -(-n // 8) * 8
        most = 819200 * 256 * 1024 // (4 if train else 1)
        m = min(_log_int(rng, 1, 819200), max(1, most // (k * n)), max(1, 819200 * 1280 // ((k + n) * (4 if train else 1))))
        return {"op": op, "m": m, "k": k, "n": n, "dtype": rng.choice(["fp16", "bf16"]),
                "act": rng.choice(["none", "gelu", "relu"]), "residual": rng.random() < 0.4, "train": train}
    if op == "layer_norm":
        d = _log_int(rng, 8, 8192)
        if rng.random() < 0.5:
            d = -(-d // 8) * 8
        rows = min(_log_int(rng, 1, 819200), max(1, 819200 * 256 // (d * (4 if train else 1))))
        return {"op": op, "rows": rows, "d": d, "dtype": rng.choice(["fp16", "bf16", "fp32"]), "train": train}
    d = _log_int(rng, 8, 768)
    if rng.random() < 0.7:
        d = -(-d // 8) * 8
    n, v = _log_int(rng, 1, 8192), _log_int(rng, 2, 200000)
    n = min(n, max(1, 8192 * 200000 * 256 // (v * d)))
    return {"op": op, "n": n, "v": v, "d": d, "dtype": rng.choice(["fp16", "bf16"]), "train": train}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dt)

    def uniform(*shape, half):
        return ((torch.rand(shape, generator=gen, device="cuda") * 2 - 1) * half).to(dt)

    s = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = normal(m, k)  # what a layer norm leaves
        s["w"], s["b"] = uniform(n, k, half=k ** -0.5), uniform(n, half=k ** -0.5)
        s["residual"] = normal(m, n) if case["residual"] else None
        if case["train"]:
            s["g"] = normal(m, n, std=0.02)
    elif case["op"] == "layer_norm":
        rows, d = case["rows"], case["d"]
        # a residual stream: rows of different spread around means of their own
        spread = 0.5 + torch.rand((rows, 1), generator=gen, device="cuda")
        centre = 0.3 * torch.randn((rows, 1), generator=gen, device="cuda")
        s["x"] = (torch.randn((rows, d), generator=gen, device="cuda") * spread + centre).to(dt)
        s["w"] = (1.0 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(dt)
        s["b"] = normal(d, std=0.1)
        if case["train"]:
            s["g"] = normal(rows, d, std=0.02)
    else:
        n, v, d = case["n"], case["v"], case["d"]
        bank = torch.nn.functional.normalize(torch.randn((v, d), generator=gen, device="cuda"), dim=1)
        target = torch.randint(0, v, (n,), generator=gen, device="cuda")
        q = bank[target] + torch.randn((n, d), generator=gen, device="cuda") * (0.6 * d ** -0.5)
        s["q"], s["bank"] = torch.nn.functional.normalize(q, dim=1).to(dt), bank.to(dt)
        # a few windows have no partner in the bank and take no part
        s["target"] = torch.where(torch.rand(n, generator=gen, device="cuda") < 0.03, torch.full_like(target, -1), target)
        if case["train"]:  # the mean's gradient; fp16 training scales its loss
            factor = 65536.0 if case["dtype"] == "fp16" else 1.0
            s["g"] = torch.full((n,), factor / n, device="cuda")
    if case["train"]:
        for name in ("x", "w", "b", "residual", "q", "bank"):
            if s.get(name) is not None:
                s[name].requires_grad_()
    return s


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        return PLAIN[case["op"]](case, state)


def _run_own(case, s):
    import neurosamble_b200  # noqa: F401
    ops = torch.ops.rbq
    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "linear":
            leaves = {"x": s["x"], "w": s["w"], "b": s["b"]}
            if case["residual"]:
                leaves["residual"] = s["residual"]
            out = {"y": ops.linear(s["x"], s["w"], s["b"], s["residual"], case["act"])}
            first = out["y"]
        elif case["op"] == "layer_norm":
            leaves = {"x": s["x"], "w": s["w"], "b": s["b"]}
            y, mean, rstd = ops.layer_norm(s["x"], s["w"], s["b"], EPS)
            out, first = {"y": y, "mean": mean, "rstd": rstd}, y
        else:
            leaves = {"q": s["q"], "bank": s["bank"]}
            loss, lse = ops.softmax_loss(s["q"], s["bank"], s["target"], SCALE)
            out, first = {"loss": loss, "lse": lse}, loss
        if case["train"]:
            grads = torch.autograd.grad(first, list(leaves.values()), s["g"])
            out.update({"d" + name: g for name, g in zip(leaves, grads)})
    return {name: t.detach() for name, t in out.items()}


def _plain_linear(case, s):
    dt = DTYPES[case["dtype"]]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t() + s["b"].float()
    if case["act"] == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * 2 ** -0.5))
        y = z * cdf
    elif case["act"] == "relu":
        y = z.clamp(min=0.0)
    else:
        y = z
    if case["residual"]:
        y = y + s["residual"].float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dz = s["g"].float()
        if case["act"] == "gelu":
            dz = dz * (cdf + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5)
        elif case["act"] == "relu":
            dz = torch.where(z > 0, dz, torch.zeros_like(dz))
        out["dx"], out["dw"], out["db"] = (dz @ w).to(dt), (dz.t() @ x).to(dt), dz.sum(0).to(dt)
        if case["residual"]:
            out["dresidual"] = s["g"].clone()
    return out


def _plain_layer_norm(case, s):
    dt = DTYPES[case["dtype"]]
    x, w = s["x"].float(), s["w"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = (c.square().mean(1, keepdim=True) + EPS).rsqrt()
    xhat = c * rstd
    out = {"y": (xhat * w + s["b"].float()).to(dt), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if case["train"]:
        g = s["g"].float()
        gw = g * w
        a, b = gw.mean(1, keepdim=True), (gw * xhat).mean(1, keepdim=True)
        out["dx"] = ((gw - a - xhat * b) * rstd).to(dt)
        out["dw"], out["db"] = (g * xhat).sum(0).to(dt), g.sum(0).to(dt)
    return out


def _plain_softmax_loss(case, s):
    dt = DTYPES[case["dtype"]]
    q, bank, target = s["q"].float(), s["bank"].float(), s["target"]
    logits = (q @ bank.t()) * SCALE
    valid = (target >= 0)[:, None]
    at = target.clamp(min=0)[:, None]
    own_logit = logits.gather(1, at)
    # the target apart from the others: the loss of a row that has learnt its target is the small
    # number log(1 + sum_others / e^target), which a difference of two near numbers would lose
    others = logits.scatter(1, at, torch.where(valid, torch.full_like(own_logit, -math.inf), own_logit))
    top = others.max(1, keepdim=True).values
    rest = top + torch.exp(others - top).sum(1, keepdim=True).log()
    u = rest - own_logit
    loss = torch.where(valid, u.clamp(min=0.0) + torch.log1p(torch.exp(-u.abs())), torch.zeros_like(u))
    lse = torch.where(valid, own_logit + loss, rest)
    out = {"loss": loss[:, 0], "lse": lse[:, 0]}
    if case["train"]:
        p = torch.exp(others - lse).scatter(1, at, torch.expm1(-loss))
        p = p * torch.where(valid, s["g"][:, None] * SCALE, torch.zeros_like(lse))
        out["dq"], out["dbank"] = (p @ bank).to(dt), (p.t() @ q).to(dt)
    return out


PLAIN = {"linear": _plain_linear, "layer_norm": _plain_layer_norm, "softmax_loss": _plain_softmax_loss}


def work(case):
    e, train = BYTES[case["dtype"]], case["train"]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        values = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        if train:  # the gradient in; those of x, w, b and the residual out
            values += m * n + m * k + n * k + n + (m * n if case["residual"] else 0)
        return {"bytes": e * values, "flops": 2 * m * n * k * (3 if train else 1)}
    if case["op"] == "layer_norm":
        rows, d = case["rows"], case["d"]
        values = 2 * rows * d + 2 * d + (2 * rows * d + 2 * d if train else 0)
        return {"bytes": e * values + 8 * rows, "flops": rows * d * (20 if train else 8)}
    n, v, d = case["n"], case["v"], case["d"]
    values = (n + v) * d * (2 if train else 1)
    return {"bytes": e * values + n * (8 + 8 + (4 if train else 0)), "flops": 2 * n * v * d * (3 if train else 1)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        s = {name: t.detach().double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for name, t in s.items()}
        return EXACT[case["op"]](case, s)


def _exact_linear(case, s):
    z = torch.einsum("mk,nk->mn", s["x"], s["w"]).add_(s["b"])
    act = {"gelu": lambda t: t * torch.special.ndtr(t), "relu": torch.relu, "none": lambda t: t}[case["act"]]
    y = act(z)
    out = {"y": y if s["residual"] is None else y + s["residual"]}
    if case["train"]:
        slope = {"gelu": lambda t: torch.special.ndtr(t) + t * torch.exp(-t.square() / 2) / math.sqrt(2 * math.pi),
                 "relu": lambda t: (t > 0).double(), "none": torch.ones_like}[case["act"]]
        dz = s["g"] * slope(z)
        out.update(dx=torch.einsum("mn,nk->mk", dz, s["w"]), dw=torch.einsum("mn,mk->nk", dz, s["x"]),
                   db=torch.einsum("mn->n", dz))
        if s["residual"] is not None:
            out["dresidual"] = s["g"]
    return out


def _exact_layer_norm(case, s):
    x, d = s["x"], case["d"]
    var, mean = torch.var_mean(x, dim=1, unbiased=False)
    rstd = 1.0 / torch.sqrt(var + EPS)
    unit = (x - mean[:, None]) * rstd[:, None]
    out = {"y": torch.addcmul(s["b"], unit, s["w"]), "mean": mean, "rstd": rstd}
    if case["train"]:
        h = s["g"] * s["w"]
        inner = d * h - h.sum(1, keepdim=True) - unit * torch.einsum("rd,rd->r", h, unit)[:, None]
        out.update(dx=inner * rstd[:, None] / d, dw=torch.einsum("rd,rd->d", s["g"], unit), db=s["g"].sum(0))
    return out


def _exact_softmax_loss(case, s):
    q, bank, target = s["q"], s["bank"], s["target"]
    n, train = case["n"], case["train"]
    lse, loss = torch.empty(n, dtype=torch.float64, device=q.device), torch.zeros(n, dtype=torch.float64, device=q.device)
    dq, dbank = torch.zeros_like(q), torch.zeros_like(bank)
    step = max(1, (1 << 28) // case["v"])
    for a in range(0, n, step):  # rows are independent but for the bank's gradient
        logits = SCALE * (q[a:a + step] @ bank.t())
        t = target[a:a + step]
        rows = torch.nonzero(t >= 0)[:, 0]
        lse[a:a + step] = torch.logsumexp(logits, 1)
        loss[a + rows] = lse[a + rows] - logits[rows, t[rows]]
        if train:
            weight = torch.zeros(t.shape[0], dtype=torch.float64, device=q.device)
            weight[rows] = SCALE * s["g"][a + rows]
            d = torch.softmax(logits, 1)
            d[rows, t[rows]] -= 1.0
            d *= weight[:, None]
            dq[a:a + step] = d @ bank
            dbank += d.t() @ q[a:a + step]
    return {"loss": loss, "lse": lse, **({"dq": dq, "dbank": dbank} if train else {})}


EXACT = {"linear": _exact_linear, "layer_norm": _exact_layer_norm, "softmax_loss": _exact_softmax_loss}
