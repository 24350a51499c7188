"""Corners of the read encoder's operators that tests/test_encoder_ops.py does not reach; the definitions in 64
bits and the tolerances are those of that file."""
import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as fw

from test_encoder_ops import (ADD, BF16, F16, F32, check_device, linear_check, linear_inputs, loss_inputs,
                              norm_check, norm_inputs, ops, tiny, u, within)


def meta(*s, dt=F16):
    return torch.empty(*s, dtype=dt, device="meta")


def forwards():
    """Each operator as a function of its differentiable inputs, with meta tensors for them (shapes only), and the
    number of inputs that its gradients read."""
    o, t = ops(), meta(4, dt=torch.int64)
    return [(lambda x, w, b, r: o.linear(x, w, b, r, "gelu"), [meta(4, 16), meta(8, 16), meta(8), meta(4, 8)], 3),
            (lambda x, w, b: o.layer_norm(x, w, b)[0], [meta(4, 16), meta(16), meta(16)], 2),
            (lambda q, k: o.softmax_loss(q, k, t, 2.0)[0], [meta(4, 16), meta(9, 16)], 2)]


# -- on the CPU -------------------------------------------------------------------------------------
def test_forward_mode_derivatives_are_refused():
    """A tangent on any input, with and without gradients, and one on the gradient that goes back."""
    for call, args, _ in forwards():
        for i in range(len(args)):
            for leaf in (False, True):
                with fw.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    primal = args[i].detach().clone().requires_grad_(leaf)
                    call(*args[:i], fw.make_dual(primal, torch.empty_like(args[i])), *args[i + 1:])
            with fw.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(*args[:i], fw.make_dual(args[i], torch.empty_like(args[i])), *args[i + 1:])
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.func.jvp(call, tuple(args), tuple(torch.empty_like(a) for a in args))
        leaves = [a.detach().clone().requires_grad_() for a in args]
        with fw.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
            y = call(*leaves)
            torch.autograd.grad(y, leaves, fw.make_dual(torch.empty_like(y), torch.empty_like(y)))
        assert call(*leaves).requires_grad  # plain calls go on


def test_second_derivatives_are_refused_on_every_way_back():
    """From each gradient to each input and to the gradient that went back, alone and beside a term that can be
    differentiated: no part of a second derivative is taken as zero."""
    for call, args, read in forwards():
        leaves = [a.detach().clone().requires_grad_() for a in args]
        y = call(*leaves)
        g = torch.empty_like(y).requires_grad_()
        grads = torch.autograd.grad(y, leaves, g, create_graph=True)
        if len(args) == 4:  # the residual's gradient is g itself
            assert torch.autograd.grad(grads[3].sum(), g, retain_graph=True)[0].shape == g.shape
            grads = grads[:3]
        for d in grads:
            assert d.requires_grad
            for t in (*leaves[:read], g):
                for out in (d.sum(), d.sum() + t.sum()):
                    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
                        torch.autograd.grad(out, t, retain_graph=True)
            with pytest.raises(RuntimeError, match="cannot be differentiated again"):
                (d.sum() + leaves[0].sum()).backward(retain_graph=True)
        plain = torch.autograd.grad(call(*leaves), leaves, g.detach())
        assert not any(d.requires_grad for d in plain)


def test_backward_operators_called_directly_refuse_more_derivatives():
    o, t = ops(), meta(4, dt=torch.int64)
    per_row = lambda: meta(4, dt=F32)  # noqa: E731
    for call, args in [
        (lambda g, x, w, b: o.linear_backward(g, x, w, b, "gelu", True, True, True), [meta(4, 8), meta(4, 16), meta(8, 16), meta(8)]),
        (lambda g, x, w, m, r: o.layer_norm_backward(g, x, w, m, r, True, True, True),
         [meta(4, 16), meta(4, 16), meta(16), per_row(), per_row()]),
        (lambda g, q, k, a, b: o.softmax_loss_backward(g, q, k, t, a, b, 2.0, True, True),
         [per_row(), meta(4, 16), meta(9, 16), per_row(), per_row()]),
    ]:
        for i in range(len(args)):
            with fw.dual_level(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(*args[:i], fw.make_dual(args[i], torch.empty_like(args[i])), *args[i + 1:])
            leaf = args[i].detach().clone().requires_grad_()
            for d in call(*args[:i], leaf, *args[i + 1:]):
                with pytest.raises(RuntimeError, match="cannot be differentiated again"):
                    torch.autograd.grad(d.sum() + leaf.sum(), leaf, retain_graph=True)
        assert not any(d.requires_grad for d in call(*args))


def strided_calls(device):
    """Every operator on inputs whose rows are not dense (transposed, sliced, expanded)."""
    o = ops()
    e = lambda *s, dt=F16: torch.zeros(*s, dtype=dt, device=device)  # noqa: E731
    x, w, g = e(2, 16, 6).transpose(1, 2), e(16, 8).t(), e(2, 8, 6).transpose(1, 2)
    row, rows, t = e(32)[::2], e(3, 2, dt=F32).t(), e(8, dt=torch.int64)[::2]
    xs, bank, each = e(16, 4).t(), e(16, 9).t(), e(1, dt=F32).expand(4)
    xn, gn = e(2, 16, 3).transpose(1, 2), e(2, 16, 3).transpose(1, 2)
    yield o.linear(x, w, e(16)[::2], g, "gelu")
    yield from o.linear_backward(g, x, w, e(16)[::2], "gelu", True, True, True)
    yield from o.layer_norm(xn, row, row)
    yield from o.layer_norm_backward(gn, xn, row, rows, rows, True, True, True)
    yield from o.softmax_loss(xs, bank, t, 2.0)
    yield from o.softmax_loss_backward(each, xs, bank, t, each, each, 2.0, True, True)


def test_meta_outputs_are_dense():
    for t in strided_calls("meta"):
        assert t.is_contiguous(), (t.shape, t.stride())


def refusals(device):
    """Calls that every device refuses, with what the message says."""
    o = ops()
    e = lambda *s, dt=F16: torch.zeros(s, dtype=dt, device=device)  # noqa: E731
    x, w, y, t, f = e(4, 16), e(8, 16), e(4, 8), e(4, dt=torch.int64), e(4, dt=F32)
    yes = (True, True, True)
    return [
        (lambda: o.linear(x.float(), w.float()), "float16 or torch.bfloat16"),
        (lambda: o.linear(x, w.bfloat16()), "w must be torch.float16"),
        (lambda: o.linear(x, e(8, 17)), r"x \[..., k\] and w \[n, k\]"),
        (lambda: o.linear(e(), w), r"x \[..., k\] and w \[n, k\]"),
        (lambda: o.linear(x, w[0]), r"x \[..., k\] and w \[n, k\]"),
        (lambda: o.linear(x, w, w[0]), "bias must have shape"),
        (lambda: o.linear(x, w, None, x), "residual must have shape"),
        (lambda: o.linear(x, w, None, None, "tanh"), "act must be one of"),
        (lambda: o.linear_backward(x, x, w, None, "none", *yes), "g must have shape"),
        (lambda: o.linear_backward(y.float(), x, w, None, "none", *yes), "g must be torch.float16"),
        (lambda: o.layer_norm(e(), w[0], w[0]), r"layer_norm takes x \[..., d\]"),
        (lambda: o.layer_norm(x, w[0, :8], w[0]), "w must have shape"),
        (lambda: o.layer_norm(x, w[0], w[0, :8]), "b must have shape"),
        (lambda: o.layer_norm(x, w[0], w[0].float()), "b must be torch.float16"),
        (lambda: o.layer_norm(x, w[0].double(), w[0].double()), "w must be torch.float16 or torch.float32"),
        (lambda: o.layer_norm_backward(y, x, w[0], f, f, *yes), "g must have shape"),
        (lambda: o.layer_norm_backward(x, x, w[0], f[:2], f, *yes), "mean must have shape"),
        (lambda: o.layer_norm_backward(x, x, w[0], f, f.half(), *yes), "rstd must be torch.float32"),
        (lambda: o.softmax_loss(x, e(8, 17), t, 1.0), "softmax_loss takes"),
        (lambda: o.softmax_loss(x[None], w, t, 1.0), "softmax_loss takes"),
        (lambda: o.softmax_loss(x, w, t.int(), 1.0), "target must be torch.int64"),
        (lambda: o.softmax_loss(x, w, t[:2], 1.0), "target must have shape"),
        (lambda: o.softmax_loss_backward(f[:2], x, w, t, f, f, 1.0, True, True), "g must have shape"),
        (lambda: o.softmax_loss_backward(f, x, w, t, f, f.half(), 1.0, True, True), "lse must be torch.float32"),
    ]


def test_meta_tensors_are_checked():
    for call, what in refusals("meta"):
        with pytest.raises(RuntimeError, match=what):
            call()


def test_errors_of_the_kernels_are_raised(monkeypatch):
    """A failed wait that the library reports (its status is planted here, on the host) becomes a RuntimeError."""
    from neurosamble_b200 import _lib, torch_ops

    class Library:
        @staticmethod
        def rbq_check_op_errors():
            return 2

        @staticmethod
        def rbq_last_error():
            return b"a tensor-core pipeline wait timed out on the device"

    monkeypatch.setattr(_lib, "lib", lambda: Library)
    with pytest.raises(RuntimeError, match="timed out"):
        torch_ops.check_op_errors()


# -- on the GPU -------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,act", [(20000, 64, 517, "gelu"), (13331, 40, 1279, "relu"), (40001, 24, 333, "gelu")])
def test_gradient_of_odd_widths_whose_last_tile_is_half_empty(m, k, n, act):
    """Rows that no TMA can read, on SM pairs of which the last one's second half has no rows (m mod 256 in
    1..128): that half stores nothing for its tile, and the staging buffers of the tiles around it are
    still waited for.  A buffer taken too early shows in one call of many, so calls repeat bit for bit."""
    x, w, b, _, g = linear_inputs(m, k, n, F16, seed=m)
    assert 1 <= m % 256 <= 128 and n % 8
    linear_check(x, w, b, None, act, g * 0.05)
    first = ops().linear_backward(g, x, w, b, act, True, True, True)
    for _ in range(20):
        assert all(torch.equal(p, q) for p, q in zip(first, ops().linear_backward(g, x, w, b, act, True, True, True)))
    check_device()


def loss_gradients(q, bank, target, g, scale=3.0):
    leaves = [q.detach().clone().requires_grad_(), bank.detach().clone().requires_grad_()]
    return torch.autograd.grad(ops().softmax_loss(*leaves, target, scale)[0], leaves, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_softmax_loss_weight_that_is_not_finite(bad, dt):
    """An infinite or NaN weight spoils its own row of dq and the bank's gradient, where the definition has
    sums of infinities, and leaves the bits of every other row's dq."""
    q, bank, target, g = loss_inputs(300, 500, 64, dt, ignored=0.1, seed=2)
    target[7] = 30
    g[7] = 0.0
    want, _ = loss_gradients(q, bank, target, g)
    g[7] = bad
    dq, dbank = loss_gradients(q, bank, target, g)
    keep = torch.arange(300, device="cuda") != 7
    assert torch.equal(dq[keep], want[keep]) and want.isfinite().all()
    assert dq[7].isnan().all() and not dbank.isfinite().any()
    g.zero_()
    g[7] = bad  # no finite weight but zeros
    dq, _ = loss_gradients(q, bank, target, g)
    assert not dq[keep].any() and dq[7].isnan().all()
    target[7] = -1  # and one of a row that takes no part
    dq, dbank = loss_gradients(q, bank, target, g)
    assert not dq.any() and not dbank.any()
    check_device()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("n,v,d", [(300, 500, 64), (70, 129, 33)])
def test_softmax_loss_rows_that_take_no_part_hold_anything(n, v, d, dt):
    """Infinities and NaN in the queries of ignored rows reach neither dq nor dbank."""
    q, bank, target, g = loss_inputs(n, v, d, dt, ignored=0.0, seed=n)
    target[5], target[6], target[n - 1] = -1, v, -100
    want = loss_gradients(q, bank, target, g)
    q[5], q[6, 3], q[n - 1] = float("nan"), float("inf"), -float("inf")
    got = loss_gradients(q, bank, target, g)
    assert all(a.isfinite().all() and torch.equal(a, b) for a, b in zip(want, got))
    got = loss_gradients(q, bank, torch.full_like(target, -1), g)
    assert not got[0].any() and not got[1].any()
    check_device()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("d", [5, 8, 40, 256, 771, 2048, 5001, 8192, 40000])
def test_layer_norm_rows_with_infinities(d, dt):
    """mean and rstd of rows with an infinity, with two of either sign and with a NaN are those of the definition at
    every width; the other rows keep their bits."""
    x = torch.randn((9, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(d)).to(dt)
    w, b = torch.full((d,), 2.0, dtype=dt, device="cuda"), torch.ones(d, dtype=dt, device="cuda")
    plain = ops().layer_norm(x, w, b)
    x[2, 1], x[3, 0], x[5, 1], x[5, 2], x[7, 3] = float("inf"), -float("inf"), float("inf"), -float("inf"), float("nan")
    y, mean, rstd = ops().layer_norm(x, w, b)
    keep = [0, 1, 4, 6, 8]
    assert all(torch.equal(a[keep], c[keep]) for a, c in zip((y, mean, rstd), plain))
    bad = [2, 3, 5, 7]
    want = x.double().mean(1)[bad].float()
    assert torch.equal(mean[bad].nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(mean[bad].isnan(), want.isnan())
    assert y[bad].isnan().all() and rstd[bad].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 256, 771, 40000])
def test_layer_norm_sums_that_overflow(d):
    """Values whose squares add up to infinity in 32 bits: rstd is 0 and y = b, as in the formula in 32 bits."""
    x = torch.randn((4, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    x[1] *= 1e25
    w, b = torch.ones(d, device="cuda"), torch.arange(d, device="cuda") / d
    y, mean, rstd = ops().layer_norm(x, w, b)
    assert rstd[1] == 0 and torch.equal(y[1], b) and mean[1].isfinite()
    assert y.isfinite().all() and (rstd[[0, 2, 3]] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
def test_gelu_keeps_its_tails(dt):
    """Value and slope of GELU at every 16-bit z in [-13.1, 13.1], through a one-wide layer whose products are
    exact: two roundings of the result, one for the output's own and one for everything before it, down to
    fp16's subnormal values (two of their roundings) and bf16's smallest normal value."""
    z = torch.arange(-2 ** 15, 2 ** 15, device="cuda").to(torch.int16).view(dt)
    z = z[z.double().abs() <= 13.1].sort().values[:, None]
    leaf = z.clone().requires_grad_()
    y = ops().linear(leaf, torch.ones(1, 1, dtype=dt, device="cuda"), None, None, "gelu")
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    check_device()
    z = z.double()
    w = z.abs()
    gauss, mills = torch.exp(-0.5 * w * w), 0.5 * torch.special.erfcx(w / math.sqrt(2))  # Phi(-w) = gauss * mills
    tail, fall = gauss * mills * w, gauss * (mills - w / math.sqrt(2 * math.pi))
    few = 2 * tiny(F16) if dt == F16 else torch.finfo(dt).smallest_normal
    for got, want, name in ((y, torch.where(z > 0, z - tail, -tail), "y"),
                            (dx, torch.where(z > 0, 1 - fall, fall), "slope")):
        within(got, want, 2 * u(dt) * want.abs() + few, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
def test_gelu_far_out(dt):
    """Infinities, NaN and the types' largest values: z or 0, and a slope of 1 or 0."""
    big = torch.finfo(dt).max
    z = torch.tensor([float("inf"), big, 14.0, 100.0, -float("inf"), -big, -14.0, -100.0, float("nan"), 0.0], device="cuda")
    z = z.to(dt)[:, None]
    leaf = z.clone().requires_grad_()
    y = ops().linear(leaf, torch.ones(1, 1, dtype=dt, device="cuda"), None, None, "gelu")
    dx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.equal(y[:4], z[:4]) and not y[4:8].any() and y[8].isnan() and y[9] == 0
    assert (dx[:4] == 1).all() and not dx[4:8].any() and dx[8].isnan() and dx[9] == 0.5


@pytest.mark.gpu
def test_outputs_have_the_strides_that_meta_tensors_say():
    for real, fake in zip(strided_calls("cuda"), strided_calls("meta"), strict=True):
        assert real.shape == fake.shape and real.stride() == fake.stride() and real.dtype == fake.dtype
    check_device()


@pytest.mark.gpu
def test_compiler_checks_of_the_operators():
    """Schemas, fake tensors and ahead-of-time tracing of forward and backward, on strided inputs."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda").to(F16).requires_grad_()  # noqa: E731
    tests = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    o, t = ops(), torch.tensor([1, 0, 8, -1], device="cuda")
    torch.library.opcheck(o.linear, (r(2, 16, 6).transpose(1, 2), r(16, 8).t(), r(8), r(2, 6, 8), "gelu"), test_utils=tests)
    torch.library.opcheck(o.layer_norm, (r(2, 16, 3).transpose(1, 2), r(16), r(16), 1e-5), test_utils=tests)
    torch.library.opcheck(o.softmax_loss, (r(16, 4).t(), r(16, 9).t(), t, 2.0), test_utils=tests)


@pytest.mark.gpu
def test_real_tensors_are_checked_alike():
    for call, what in refusals("cuda"):
        with pytest.raises(RuntimeError, match=what):
            call()


def check_loss_gradients_by_rows(q, bank, target, scale, g, dq, dbank, rows=1024):
    """test_encoder_ops.loss_check's gradients and tolerances, `rows` queries at a time."""
    dt, (n, d), v = q.dtype, q.shape, bank.shape[0]
    K = bank.double()
    wdk, tdk = torch.zeros_like(K), torch.zeros_like(K)
    top = g[(target >= 0) & (target < v)].abs().max().double()
    for a in range(0, n, rows):
        Q, t = q[a:a + rows].double(), target[a:a + rows]
        s = scale * (Q @ K.t())
        es = (d + 8) * ADD * scale * (Q.abs() @ K.abs().t()) + 4 * ADD * s.abs()
        valid = (t >= 0) & (t < v)
        weight = torch.where(valid, g[a:a + rows].double(), torch.zeros(1, dtype=torch.float64, device=q.device))
        lse = torch.logsumexp(s, 1)
        e = es.max(1).values + (v + 64) * ADD * 2 + 4 * ADD * lse.abs()
        dl = torch.exp(s - lse[:, None])
        at = torch.arange(len(t), device=q.device)[valid]
        own = dl[at, t[valid]].clone()
        dl[at, t[valid]] = 0.0
        dl[at, t[valid]] = -dl[valid].sum(1)  # 1 - p without its cancellation
        assert (own + dl[at, t[valid]].abs() - 1).abs().max() < 1e-9
        dl *= weight[:, None]
        el = (u(dt) + 8 * ADD) * dl.abs() + 2 * (e[:, None] + es) * dl.abs() * 1.01 + (2.0 ** -38 * top if dt == F16 else 0.0)
        wdq = scale * dl @ K
        within(dq[a:a + rows], wdq, (u(dt) + 4 * ADD) * wdq.abs() + 1.01 * scale * (el + (v + 72) * ADD * dl.abs()) @ K.abs() +
               tiny(dt), f"dq from row {a}")
        wdk += scale * dl.t() @ Q
        tdk += 1.01 * scale * (el + (n + 72) * ADD * dl.abs()).t() @ Q.abs()
    within(dbank, wdk, (u(dt) + 4 * ADD) * wdk.abs() + tdk + tiny(dt), "dbank")


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,d,dt", [(8192, 80001, 40, F16), (200003, 4001, 24, BF16), (9001, 75003, 33, BF16)])
def test_softmax_loss_gradient_in_several_pieces(n, v, d, dt):
    """Banks whose logits' gradient does not fit the workspace at once: the queries' gradient is added up over the
    pieces, the bank's written piece by piece, and the last piece is shorter and odd.  It repeats bit for
    bit, alone and on two streams at once."""
    from neurosamble_b200 import _lib
    need = ctypes.c_int64()
    _lib.call("rbq_softmax_loss_workspace", n, v, d, 0 if dt == F16 else 1, 1, ctypes.byref(need))
    assert need.value < 2 * n * v  # not even the gradient of all logits
    q, bank, target, g = loss_inputs(n, v, d, dt, seed=n)
    target[:3] = torch.tensor([v - 1, v - 2, 0], device="cuda")  # in the last piece and in the first
    loss, lse = ops().softmax_loss(q, bank, target, 5.0)
    run = lambda: ops().softmax_loss_backward(g, q, bank, target, loss, lse, 5.0, True, True)  # noqa: E731
    dq, dbank = run()
    check_loss_gradients_by_rows(q, bank, target, 5.0, g, dq, dbank)
    one = ops().softmax_loss_backward(g, q, bank, target, loss, lse, 5.0, True, False)[0]
    other = ops().softmax_loss_backward(g, q, bank, target, loss, lse, 5.0, False, True)[1]
    assert torch.equal(one, dq) and torch.equal(other, dbank)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(2):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, dq) and torch.equal(b, dbank) for a, b in outs)
    check_device()


@pytest.mark.gpu
@pytest.mark.parametrize("dt,pdt", [(F16, F32), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("d", [1, 3, 7, 9, 31, 33, 65, 127, 255, 257])
def test_layer_norm_narrow_odd_rows_in_rounds(d, dt, pdt):
    """Widths that take single values, with more rows than the blocks hold at once."""
    norm_check(*norm_inputs(40001, d, dt, pdt, seed=d))


@pytest.mark.gpu
def test_no_errors_were_recorded():
    from neurosamble_b200 import torch_ops
    x = torch.ones(256, 64, dtype=F16, device="cuda")
    ops().linear(x, x)
    assert torch_ops.check_op_errors() is None


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("m,k,n", [(65, 8, 40), (1001, 8, 37), (5001, 16, 300), (20000, 8, 517)])
def test_bias_gradients_that_cancel(m, k, n, dt):
    """Bias gradients far smaller than their terms, which a last row cancels: they are sums of fp32 terms,
    rounded once, without the rounding to 16 bits that the products' operand has."""
    x, w, b, _, g = linear_inputs(m, k, n, dt, seed=m)
    w, x[-1] = w.abs(), 60.0  # the last row's slope is 1 in every column
    z = x.double() @ w.double().t() + b.double()
    slope = torch.special.ndtr(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    assert (slope[-1] == 1).all()
    g[-1] = 0
    g[-1] = -(g.double() * slope).sum(0).to(dt)
    dz = g.double() * slope
    want = dz.sum(0)
    db = ops().linear_backward(g, x, w, b, "gelu", True, True, True)[2]
    check_device()
    # an error of z's sum and of the slope (|gelu''| <= 0.8), and fp32 additions; one rounding of the result
    ez = (k + 8) * ADD * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    tol = ((0.8 * ez + 4e-6 * (1 + z.abs())) * g.double().abs() * (slope != 1)).sum(0) + (m + 8) * ADD * dz.abs().sum(0)
    within(db, want, (u(dt) + ADD) * want.abs() + 1.01 * tol + tiny(dt), "db")


@pytest.mark.gpu
@pytest.mark.parametrize("n,v,d", [(1, 512, 8), (700, 512, 40), (40, 1024, 64), (33, 1024, 33), (300, 2048, 24)])
def test_query_gradients_that_cancel(n, v, d):
    """A bank of equal rows: every probability is 1 / v, the target's entry cancels all the others and dq is 0.
    The others are powers of two, which 16 bits hold; the target's, 1 - 1 / v, takes more bits than bf16 has,
    and what its rounding leaves is not in dq."""
    q, bank, target, _ = loss_inputs(n, v, d, BF16, ignored=0.0, seed=v)
    bank, scale = bank[:1].expand(v, d).contiguous(), 4.0
    dq, _ = loss_gradients(q, bank, target, torch.ones(n, device="cuda"), scale)
    check_device()
    s = scale * (q.double() @ bank[0].double())
    es = (d + 8) * ADD * scale * (q.double().abs() @ bank[0].double().abs()) + 4 * ADD * s.abs()
    e = es + (v + 64) * ADD * 2 + 4 * ADD * (s + math.log(v)).abs()
    assert (2 * (e + es) < u(BF16) / 2).all()  # the others round to 1 / v whatever their error
    # the target's entry, expm1(-loss): the loss's error times 1 / v, and fp32; a sum of v products whose
    # magnitudes add up to 2; and the rounding of what the entry's own rounding left
    each = 2 * e / v + 8 * ADD + 2 * (v + 72) * ADD + u(BF16) ** 2
    tol = 1.01 * scale * each[:, None] * bank[0].double().abs()
    within(dq, torch.zeros_like(q, dtype=torch.float64), tol + tiny(BF16), "dq")
