"""The read encoder's operators (torch.ops.rbq.linear, layer_norm, softmax_loss) against their
definitions in 64 bits, forward and backward, and their refusals.

Tolerances follow from the arithmetic.  u = finfo(t).eps / 2 is one rounding to type t.  A sum of K
products in fp32 is off by at most (K + 8) * 2^-23 of the sum of their magnitudes (2^-23 per addition
also covers an accumulator that truncates; 8 for the few operations around the sum).  Where the
kernels round an intermediate to 16 bits (dz, and the gradient of the logits) its u is counted on
every product that reads it."""
import ctypes
import math

import numpy as np
import pytest
import torch

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ADD = 2.0 ** -23


def u(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half the distance of subnormal values: what rounding loses near zero."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def within(got, want, tol, name):
    """|got - want| <= tol; a value past the type's largest one rounds to infinity."""
    largest = torch.finfo(got.dtype).max
    got = got.detach().double()
    assert got.shape == want.shape, name
    bad = ~((got - want).abs() <= tol)
    over = want.abs() + tol > largest
    bad &= ~(over & got.isinf() & (got.sign() == want.sign()))
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float(((got - want).abs() / tol).nan_to_num(float('inf')).max()):.3g} of the tolerance")


def ops():
    import neurosamble_b200  # noqa: F401  (registers the operators)
    return torch.ops.rbq


def check_device():
    from neurosamble_b200 import _lib
    torch.cuda.synchronize()
    _lib.call("rbq_check_op_errors")


# -- on the CPU: registration, shapes, refusals ---------------------------------------------------
def meta(*s, dt=F16):
    return torch.empty(*s, dtype=dt, device="meta")


def test_registered_with_shapes():
    o = ops()
    assert o.linear(meta(5, 7, 16), meta(24, 16), meta(24), None, "gelu").shape == (5, 7, 24)
    y, mean, rstd = o.layer_norm(meta(5, 7, 16), meta(16), meta(16))
    assert y.shape == (5, 7, 16) and mean.shape == rstd.shape == (5, 7) and mean.dtype == F32
    loss, lse = o.softmax_loss(meta(5, 16), meta(9, 16), meta(5, dt=torch.int64), 10.0)
    assert loss.shape == lse.shape == (5,) and loss.dtype == F32


def test_host_tensors_are_refused():
    o = ops()
    x = torch.zeros(3, 8, dtype=F16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        o.linear(x, x)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        o.layer_norm(x, x[0], x[0])
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        o.softmax_loss(x, x, torch.zeros(3, dtype=torch.int64), 1.0)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        o.linear(x.requires_grad_(), x.detach())


@pytest.mark.gpu  # autograd's engine wants the device that the fake tensors name
def test_fake_tensors_keep_their_shapes_through_a_backward_pass():
    from torch._subclasses.fake_tensor import FakeTensorMode
    o = ops()
    with FakeTensorMode():
        x = torch.empty(6, 16, dtype=F16, device="cuda", requires_grad=True)
        w = torch.empty(24, 16, dtype=F16, device="cuda", requires_grad=True)
        y = o.linear(x, w, None, None, "relu")
        dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
        assert y.shape == (6, 24) and dx.shape == (6, 16) and dw.shape == (24, 16) and dw.device.type == "cuda"
        n = torch.empty(16, device="cuda", requires_grad=True)
        dx, dn = torch.autograd.grad(o.layer_norm(x, n, n)[0], (x, n), torch.empty_like(x))
        assert dx.dtype == F16 and dn.dtype == F32 and dn.shape == (16,)
        t = torch.empty(6, dtype=torch.int64, device="cuda")
        loss = o.softmax_loss(x, w, t, 2.0)[0]
        dq, dk = torch.autograd.grad(loss, (x, w), torch.empty_like(loss))
        assert dq.shape == (6, 16) and dk.shape == (24, 16)


P1 = ctypes.c_void_p(16)  # never dereferenced: the checks come first


@pytest.mark.parametrize("args,what", [
    ((P1, P1, None, None, P1, 4, 8, 8, 2, 0, None, 0, None), "RBQ_F16 or RBQ_BF16"),
    ((P1, P1, None, None, P1, 4, 8, 8, 0, 3, None, 0, None), "unknown activation"),
    ((P1, P1, None, None, P1, 4, 0, 8, 0, 0, None, 0, None), "bad sizes"),
    ((P1, P1, None, None, P1, -1, 8, 8, 0, 0, None, 0, None), "bad sizes"),
    ((P1, P1, None, None, P1, 2 ** 31, 8, 8, 0, 0, None, 0, None), "bad sizes"),
    ((None, P1, None, None, P1, 4, 8, 8, 0, 0, None, 0, None), "null buffer"),
    ((ctypes.c_void_p(18), P1, None, None, P1, 4, 8, 8, 0, 0, None, 0, None), "16-byte boundaries"),
])
def test_linear_refusals(args, what):
    from neurosamble_b200 import _lib
    assert _lib.lib().rbq_linear(*args) == 1
    assert what in _lib.lib().rbq_last_error().decode()


@pytest.mark.parametrize("args,what", [
    ((P1, P1, P1, P1, P1, P1, 4, 0, 1e-5, 0, 0, None), "bad sizes"),
    ((P1, P1, P1, P1, P1, P1, 4, 8, -1.0, 0, 0, None), "eps"),
    ((P1, P1, P1, P1, P1, P1, 4, 8, float("nan"), 0, 0, None), "eps"),
    ((P1, P1, P1, P1, P1, P1, 4, 8, 1e-5, 0, 1, None), "param_dtype"),
    ((P1, P1, P1, P1, P1, P1, 4, 8, 1e-5, 7, 7, None), "dtype"),
    ((P1, P1, None, P1, P1, P1, 4, 8, 1e-5, 0, 0, None), "null buffer"),
])
def test_layer_norm_refusals(args, what):
    from neurosamble_b200 import _lib
    assert _lib.lib().rbq_layer_norm(*args) == 1
    assert what in _lib.lib().rbq_last_error().decode()


@pytest.mark.parametrize("args,what", [
    ((P1, P1, P1, 4, 0, 8, 1.0, 0, P1, P1, None, 0, None), "bad sizes"),
    ((P1, P1, P1, 4, 8, 8, 0.0, 0, P1, P1, None, 0, None), "scale"),
    ((P1, P1, P1, 4, 8, 8, float("inf"), 0, P1, P1, None, 0, None), "scale"),
    ((P1, P1, P1, 4, 8, 8, float("nan"), 0, P1, P1, None, 0, None), "scale"),
    ((P1, P1, P1, 4, 8, 8, 1.0, 2, P1, P1, None, 0, None), "RBQ_F16 or RBQ_BF16"),
    ((P1, P1, None, 4, 8, 8, 1.0, 0, P1, P1, None, 0, None), "null buffer"),
])
def test_softmax_loss_refusals(args, what):
    from neurosamble_b200 import _lib
    assert _lib.lib().rbq_softmax_loss(*args) == 1
    assert what in _lib.lib().rbq_last_error().decode()


def test_empty_calls_need_no_device():
    from neurosamble_b200 import _lib
    L = _lib.lib()
    assert L.rbq_linear(None, None, None, None, None, 0, 8, 8, 0, 0, None, 0, None) == 0
    assert L.rbq_layer_norm(None, None, None, None, None, None, 0, 8, 1e-5, 0, 0, None) == 0
    assert L.rbq_softmax_loss(None, None, None, 0, 8, 8, 1.0, 0, None, None, None, 0, None) == 0
    need = ctypes.c_int64(5)
    assert L.rbq_linear_workspace(0, 8, 8, 0, 0, 1, ctypes.byref(need)) == 0 and need.value == 0


@pytest.mark.gpu
def test_wrapper_refusals():
    o = ops()
    x, w = torch.zeros(4, 16, dtype=F16, device="cuda"), torch.zeros(8, 16, dtype=F16, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for call, what in [
        (lambda: o.linear(x.float(), w.float()), "float16 or torch.bfloat16"),
        (lambda: o.linear(x, w.bfloat16()), "w must be torch.float16"),
        (lambda: o.linear(x, w[:, :8]), r"x \[..., k\] and w \[n, k\]"),
        (lambda: o.linear(x, w, w[0]), "bias must have shape"),
        (lambda: o.linear(x, w, None, x), "residual must have shape"),
        (lambda: o.linear(x, w, None, None, "tanh"), "act must be one of"),
        (lambda: o.linear(x, w.cpu()), "w must be a CUDA tensor"),
        (lambda: o.layer_norm(x, w[0, :8], w[0, :8]), "w must have shape"),
        (lambda: o.layer_norm(x, w[0].bfloat16(), w[0].bfloat16()), "w must be torch.float16 or torch.float32"),
        (lambda: o.layer_norm(x, w[0], w[0].float()), "b must be torch.float16"),
        (lambda: o.layer_norm(x, w[0].cpu(), w[0]), "w must be a CUDA tensor"),
        (lambda: o.softmax_loss(x, w.cpu(), t, 1.0), "bank must be a CUDA tensor"),
        (lambda: o.layer_norm(x, w[0], w[0], -1.0), "eps"),
        (lambda: o.softmax_loss(x, w, t.int(), 1.0), "target must be torch.int64"),
        (lambda: o.softmax_loss(x, w, t[:2], 1.0), "target must have shape"),
        (lambda: o.softmax_loss(x, w[:, :8], t, 1.0), "softmax_loss takes"),
        (lambda: o.softmax_loss(x, w[:0], t, 1.0), "softmax_loss takes"),
        (lambda: o.softmax_loss(x, w, t, -1.0), "scale"),
        (lambda: o.softmax_loss(x, w, t.cpu(), 1.0), "target must be a CUDA tensor"),
    ]:
        with pytest.raises(RuntimeError, match=what):
            call()


@pytest.mark.gpu
def test_short_workspace_is_refused():
    from neurosamble_b200 import _lib
    x = torch.zeros(64, 8, dtype=F16, device="cuda")
    t = torch.zeros(64, dtype=torch.int64, device="cuda")
    f = torch.zeros(64, device="cuda")
    p = lambda v: ctypes.c_void_p(v.data_ptr())  # noqa: E731
    st = _lib.lib().rbq_softmax_loss(p(x), p(x), p(t), 64, 64, 8, 1.0, 0, p(f), p(f), p(x), 16, None)
    assert st == 1 and "bytes" in _lib.lib().rbq_last_error().decode()


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    o = ops()
    x = torch.randn(4, 16, device="cuda").to(F16).requires_grad_()
    w = torch.randn(8, 16, device="cuda").to(F16).requires_grad_()
    y = o.linear(x, w, None, None, "gelu")
    dx, = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        dx.float().sum().backward()


# -- linear ----------------------------------------------------------------------------------------
def gelu_parts(z):
    cdf = torch.special.ndtr(z)
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def linear_check(x, w, b, res, act, g, call=None, name=""):
    """Forward and gradients of one layer; x, w, b, res, g 16-bit CUDA tensors (2-D)."""
    dt, k, n, m = x.dtype, x.shape[1], w.shape[0], x.shape[0]
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b, res) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, b, res)]
    y = (call or ops().linear)(*args, act)
    grads = dict(zip([s for s, t in zip(("x", "w", "b", "r"), (x, w, b, res)) if t is not None],
                     torch.autograd.grad(y, leaves, g)))
    check_device()
    X, W, G = x.double(), w.double(), g.double()
    B = b.double() if b is not None else torch.zeros(n, dtype=torch.float64, device=x.device)
    z = X @ W.t() + B
    ez = (k + 8) * ADD * (X.abs() @ W.abs().t() + B.abs())  # what fp32 may lose of z
    if act == "gelu":
        a, slope = gelu_parts(z)
        # |gelu'| <= 1.13 and |gelu''| <= 0.8; the kernel's Phi and phi are good to 2e-6 and 2^-9 of a rounding
        ea, es = 1.13 * ez + 2e-6 * (1 + z.abs()), 0.8 * ez + 4e-6 * (1 + z.abs())
    elif act == "relu":
        a, slope = torch.relu(z), (z > 0).double()
        ea, es = ez, (z.abs() <= ez).double()  # the sign of z is open within its error
    else:
        a, slope, ea, es = z, torch.ones_like(z), ez, torch.zeros_like(z)
    want = a if res is None else a + res.double()
    within(y, want, (u(dt) + 8 * ADD) * want.abs() + ea * (1 + u(dt)) + tiny(dt), name + "y")
    dz = G * slope
    # dz is the operand of the products: one rounding, the error of act', and fp32 around it
    round_dz = u(dt) if act != "none" else 0.0
    edz = round_dz * dz.abs() + es * G.abs() * 1.01 + 8 * ADD * dz.abs() + (tiny(dt) if act != "none" else 0.0)
    dx, dw, db = dz @ W, dz.t() @ X, dz.sum(0)
    within(grads["x"], dx, (u(dt) + ADD) * dx.abs() + 1.01 * edz @ W.abs() + (n + 8) * ADD * dz.abs() @ W.abs() + tiny(dt),
           name + "dx")
    within(grads["w"], dw, (u(dt) + ADD) * dw.abs() + 1.01 * edz.t() @ X.abs() + (m + 72) * ADD * dz.abs().t() @ X.abs() +
           tiny(dt), name + "dw")
    if b is not None:
        within(grads["b"], db, (u(dt) + ADD) * db.abs() + 1.01 * edz.sum(0) + (m + 8) * ADD * dz.abs().sum(0) + tiny(dt),
               name + "db")
    if res is not None:
        assert torch.equal(grads["r"], g)


def linear_inputs(m, k, n, dt, res=False, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    return (r(m, k).to(dt), (r(n, k) * k ** -0.5).to(dt), (0.3 * r(n)).to(dt), r(m, n).to(dt) if res else None,
            r(m, n).to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 256, 1024), (127, 64, 128), (128, 65, 136), (129, 8, 264), (400, 256, 1024),
                                   (333, 331, 517), (1000, 72, 7), (5, 513, 129), (2049, 16, 255), (300, 1024, 256)])
def test_linear(m, k, n, act, dt):
    x, w, b, _, g = linear_inputs(m, k, n, dt, seed=m * 7 + k * 3 + n)
    linear_check(x, w, b, None, act, g)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
@pytest.mark.parametrize("m,k,n", [(1, 8, 8), (400, 1024, 256), (130, 40, 333), (20000, 64, 136), (257, 257, 257)])
def test_linear_residual(m, k, n, act, dt):
    linear_check(*linear_inputs(m, k, n, dt, res=True, seed=m + n)[:4], act, linear_inputs(m, k, n, dt, seed=5)[4])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [40000, 40001])
def test_linear_many_rows(m):
    """More tiles than SMs in every product, and a weight gradient split over the rows."""
    x, w, b, res, g = linear_inputs(m, 96, 320, F16, res=True, seed=3)
    linear_check(x, w, b, res, "gelu", g * 0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("m,k,n", [(2048, 24, 4100), (2100, 40, 4104), (5000, 700, 904), (9000, 520, 72), (3000, 1500, 1480)])
def test_linear_sums_over_uneven_tiles(m, k, n, act):
    """Weight gradients whose k-blocks the CTAs share unevenly, and bias sums of columns with fewer tiles
    than there are CTAs."""
    x, w, b, _, g = linear_inputs(m, k, n, F16, seed=m + k)
    linear_check(x, w, b, None, act, g * 0.05)


@pytest.mark.gpu
def test_linear_without_bias_and_with_few_gradients():
    x, w, _, _, g = linear_inputs(200, 48, 80, BF16)
    linear_check(x, w, None, None, "gelu", g)
    o = ops()
    full = [t.clone().requires_grad_() for t in (x, w)]
    dx, dw = torch.autograd.grad(o.linear(*full, None, None, "gelu"), full, g)
    wl = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(o.linear(x, wl, None, None, "gelu"), wl, g)[0], dw)
    xl = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(o.linear(xl, w, None, None, "gelu"), xl, g)[0], dx)
    check_device()


@pytest.mark.gpu
def test_linear_gelu_over_its_range():
    """z from -12 to 12 through a one-wide layer: the value and the slope of GELU on a grid."""
    for dt in (F16, BF16):
        x = torch.linspace(-12, 12, 4801, device="cuda").to(dt)[:, None]
        one = torch.ones(1, 1, dtype=dt, device="cuda")
        linear_check(x, one, torch.zeros(1, dtype=dt, device="cuda"), None, "gelu", torch.ones_like(x))


@pytest.mark.gpu
def test_linear_strides_batches_and_views():
    """Leading dimensions, transposed weights, row slices, expanded gradients and an offset that TMA
    could not address give the dense call's bits."""
    o = ops()
    x, w, b, _, g = linear_inputs(60, 24, 40, F16)
    y = o.linear(x, w, b, None, "gelu")
    assert torch.equal(o.linear(x.view(3, 4, 5, 24), w, b, None, "gelu").view(60, 40), y)
    assert torch.equal(o.linear(x.t().contiguous().t(), w.t().contiguous().t(), b, None, "gelu"), y)
    wide = torch.zeros(60, 64, dtype=F16, device="cuda")
    wide[:, 3:27] = x
    assert torch.equal(o.linear(wide[:, 3:27], w, b, None, "gelu"), y)
    flat = torch.zeros(60 * 24 + 1, dtype=F16, device="cuda")
    flat[1:] = x.reshape(-1)
    assert torch.equal(o.linear(flat[1:].view(60, 24), w, b, None, "gelu"), y)
    xl = x.clone().requires_grad_()
    got, = torch.autograd.grad(o.linear(xl, w, b, None, "gelu").float().sum(), xl)
    want, = torch.autograd.grad(o.linear(xl, w, b, None, "gelu"), xl, torch.ones_like(y))
    assert torch.equal(got, want)
    check_device()


@pytest.mark.gpu
def test_linear_nothing_to_do():
    o = ops()
    x = torch.zeros(0, 16, dtype=F16, device="cuda", requires_grad=True)
    w = torch.ones(8, 16, dtype=F16, device="cuda", requires_grad=True)
    b = torch.ones(8, dtype=F16, device="cuda", requires_grad=True)
    y = o.linear(x, w, b, None, "gelu")
    assert y.shape == (0, 8)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert dx.shape == (0, 16) and not dw.any() and not db.any()


@pytest.mark.gpu
def test_linear_infinities_and_nan_stay_in_their_rows():
    o = ops()
    x, w, b, _, _ = linear_inputs(300, 40, 50, BF16)
    y = o.linear(x, w, b, None, "relu")
    x[7, 3], x[200, 0] = float("nan"), float("inf")
    z = o.linear(x, w, b, None, "relu")
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[7] = keep[200] = False
    assert torch.equal(z[keep], y[keep]) and z[7].isnan().all()
    want = torch.relu(x[200].double() @ w.double().t() + b.double())
    assert torch.equal(z[200].isinf(), want.isinf()) and not z[200].isnan().any()


@pytest.mark.gpu
def test_linear_leaves_what_lies_behind_its_output():
    from neurosamble_b200 import _lib
    p = lambda v: ctypes.c_void_p(v.data_ptr())  # noqa: E731
    for m, n in ((130, 136), (130, 133)):
        x, w, b, _, _ = linear_inputs(m, 16, n, F16)
        buf = torch.full((m * n + 4096,), 7.0, dtype=F16, device="cuda")
        _lib.call("rbq_linear", p(x), p(w), p(b), None, p(buf), m, 16, n, 0, 2, None, 0,
                  ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        check_device()
        assert torch.equal(buf[:m * n].view(m, n), ops().linear(x, w, b, None, "gelu"))
        assert (buf[m * n:] == 7.0).all()


# -- layer norm ------------------------------------------------------------------------------------
def norm_check(x, w, b, g, eps=1e-5, name=""):
    dt, pdt, d, rows = x.dtype, w.dtype, x.shape[1], x.shape[0]
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    y, mean, rstd = ops().layer_norm(*leaves, eps)
    assert not mean.requires_grad and not rstd.requires_grad
    dx, dw, db = torch.autograd.grad(y, leaves, g)
    torch.cuda.synchronize()
    X, W, B, G = x.double(), w.double(), b.double(), g.double()
    mu = X.mean(1, keepdim=True)
    c = X - mu
    r = 1.0 / torch.sqrt(c.square().mean(1, keepdim=True) + eps)
    h = c * r
    want = h * W + B
    # the mean is a sum of d values; a difference from it carries its error, and the two-pass variance
    # twice the relative error of the differences, halved by the root
    emu = (d + 8) * ADD * X.abs().mean(1, keepdim=True)
    ec = emu + ADD * c.abs()
    rel_r = (d + 16) * ADD + r * r * (c.abs() * ec * 2 + ec * ec).mean(1, keepdim=True)
    eh = ec * r + h.abs() * rel_r + 4 * ADD * h.abs()
    within(mean[:, None], mu, emu + ADD * mu.abs(), name + "mean")
    within(rstd[:, None], r, (rel_r + 8 * ADD) * r, name + "rstd")
    within(y, want, (u(dt) + 4 * ADD) * want.abs() + eh * W.abs() * 1.01 + 4 * ADD * (h * W).abs() + tiny(dt), name + "y")
    gw = G * W
    ea, ebh = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
    wdx = r * (gw - ea - h * ebh)
    sums = gw.abs().mean(1, keepdim=True)
    hs = (gw * h).abs().mean(1, keepdim=True)
    err = (d + 8) * ADD * sums + h.abs() * ((d + 8) * ADD * hs + (gw.abs() * eh).mean(1, keepdim=True)) + eh * ebh.abs()
    err = r * (err + 8 * ADD * (gw.abs() + ea.abs() + (h * ebh).abs())) + rel_r * wdx.abs()
    within(dx, wdx, (u(dt) + 4 * ADD) * wdx.abs() + 1.01 * err + tiny(dt), name + "dx")
    wdw, wdb = (G * h).sum(0), G.sum(0)
    within(dw, wdw, (u(pdt) + ADD) * wdw.abs() + (rows + 64) * ADD * (G * h).abs().sum(0) + 1.01 * (G.abs() * eh).sum(0) +
           tiny(pdt), name + "dw")
    within(db, wdb, (u(pdt) + ADD) * wdb.abs() + (rows + 64) * ADD * G.abs().sum(0) + tiny(pdt), name + "db")


def norm_inputs(rows, d, dt, pdt, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    x = (r(rows, d) * (0.5 + torch.rand((rows, 1), generator=gen, device="cuda")) + r(rows, 1)).to(dt)
    return x, (1 + 0.3 * r(d)).to(pdt), r(d).to(pdt), r(rows, d).to(dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,pdt", [(F16, F16), (F16, F32), (BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("rows,d", [(1, 8), (1, 256), (3, 5), (400, 256), (1001, 40), (77, 23), (130, 512), (65, 771),
                                    (64, 1024), (33, 1032), (17, 8192), (9, 5001), (5, 40000), (4, 40001), (3000, 64)])
def test_layer_norm(rows, d, dt, pdt):
    norm_check(*norm_inputs(rows, d, dt, pdt, seed=rows + d))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,pdt", [(F16, F32), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("d", [1000, 1023, 1025, 1953, 2048, 2049, 4095, 4096, 4104, 8192, 8200])
def test_layer_norm_wide_rows_in_rounds(d, dt, pdt):
    """Rows held by a whole block, of every number of loads per thread, and blocks that take several."""
    norm_check(*norm_inputs(2999, d, dt, pdt, seed=d))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [1, 2, 8])
def test_layer_norm_rows_without_spread(d):
    """Equal values: variance 0, y = b, and a gradient of the size of 1 / sqrt(eps)."""
    for dt in (F16, F32):
        x = torch.full((5, d), 3.0, dtype=dt, device="cuda")
        w, b = torch.ones(d, dtype=dt, device="cuda"), torch.arange(d, device="cuda").to(dt)
        norm_check(x, w, b, torch.randn(5, d, device="cuda").to(dt) * 0.01)


@pytest.mark.gpu
def test_layer_norm_far_mean():
    """A mean far above the spread: the two-pass variance keeps it."""
    x = (1000 + torch.randn(300, 256, device="cuda"))
    norm_check(x, torch.ones(256, device="cuda"), torch.zeros(256, device="cuda"), torch.randn(300, 256, device="cuda"))


@pytest.mark.gpu
def test_layer_norm_many_rows_and_views():
    norm_check(*norm_inputs(30011, 256, BF16, F32, seed=9))
    o = ops()
    x, w, b, g = norm_inputs(60, 48, F16, F16)
    y, mean, rstd = o.layer_norm(x, w, b)
    y2, mean2, _ = o.layer_norm(x.view(3, 20, 48), w, b)
    assert torch.equal(y2.view(60, 48), y) and torch.equal(mean2.view(60), mean)
    assert torch.equal(o.layer_norm(x.t().contiguous().t(), w, b)[0], y)
    pad = torch.zeros(49, dtype=F16, device="cuda")
    pad[1:] = w  # parameters off the 16-byte boundary: loads of one value, the same arithmetic
    norm_check(x, pad[1:], b, g)
    leaf = x.clone().requires_grad_()
    got, = torch.autograd.grad(o.layer_norm(leaf, w, b)[0].sum(), leaf)
    want, = torch.autograd.grad(o.layer_norm(leaf, w, b)[0], leaf, torch.ones_like(x))
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_layer_norm_nothing_to_do_and_nan():
    o = ops()
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y, mean, _ = o.layer_norm(x, w, w)
    assert y.shape == (0, 16) and mean.shape == (0,)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == (0, 16) and not dw.any()
    x, w, b, _ = norm_inputs(50, 40, F16, F16)
    y = o.layer_norm(x, w, b)[0]
    x[3, 1], x[40, 2] = float("nan"), float("inf")
    z = o.layer_norm(x, w, b)[0]
    keep = torch.ones(50, dtype=torch.bool, device="cuda")
    keep[3] = keep[40] = False
    assert torch.equal(z[keep], y[keep]) and z[3].isnan().all() and z[40].isnan().all()


# -- softmax loss ----------------------------------------------------------------------------------
def loss_check(q, bank, target, scale, g, name=""):
    dt, (n, d), v = q.dtype, q.shape, bank.shape[0]
    leaves = [t.detach().clone().requires_grad_() for t in (q, bank)]
    loss, lse = ops().softmax_loss(*leaves, target, scale)
    assert not lse.requires_grad
    dq, dbank = torch.autograd.grad(loss, leaves, g)
    check_device()
    Q, K, G = q.double(), bank.double(), g.double()
    s = scale * (Q @ K.t())
    valid = (target >= 0) & (target < v)
    at = target.clamp(0, v - 1)[:, None]
    wlse = torch.logsumexp(s, 1)
    others = s.scatter(1, at, torch.where(valid[:, None], torch.full_like(s[:, :1], -math.inf), s.gather(1, at)))
    rest = torch.logsumexp(others, 1)
    own = s.gather(1, at)[:, 0]
    wloss = torch.where(valid, torch.nn.functional.softplus(rest - own, threshold=200.0), torch.zeros_like(own))
    # a logit's error: the product's sum, and the rounding of scale * log2(e) and of its exponent
    es = (d + 8) * ADD * scale * (Q.abs() @ K.abs().t()) + 4 * ADD * s.abs()
    # sums of exponentials: v values, the worst logit's error, 2^-22 for each exponential
    e = es.max(1).values + (v + 64) * ADD * 2 + 4 * ADD * wlse.abs().clamp(max=1e6)
    p_rest = torch.where(valid, torch.sigmoid(rest - own), torch.zeros_like(own))
    within(loss, wloss, 2 * p_rest * e + 4 * ADD * wloss + tiny(F32), name + "loss")
    within(lse, wlse, 2 * e + 4 * ADD * wlse.abs() + tiny(F32), name + "lse")
    p = torch.softmax(s, 1)
    dl = p.clone()
    rows = torch.arange(n, device=q.device)[valid]
    dl[rows, target[valid]] = torch.expm1(-wloss[valid])
    weight = torch.where(valid, G, torch.zeros_like(G))[:, None]
    dl = dl * weight
    top = weight.abs().max()
    # one rounding to the operands' type, relative to the value down to 2^-28 of the largest weight
    # (fp16 subnormals: half of 2^-24, over the scale of at least 2^13), and the probability's error
    el = (u(dt) + 8 * ADD) * dl.abs() + 2 * (e[:, None] + es) * dl.abs() * 1.01 + (2.0 ** -38 * top if dt == F16 else 0.0)
    wdq, wdk = scale * dl @ K, scale * dl.t() @ Q
    within(dq, wdq, (u(dt) + 4 * ADD) * wdq.abs() + 1.01 * scale * (el + (v + 72) * ADD * dl.abs()) @ K.abs() + tiny(dt),
           name + "dq")
    within(dbank, wdk, (u(dt) + 4 * ADD) * wdk.abs() + 1.01 * scale * (el + (n + 72) * ADD * dl.abs()).t() @ Q.abs() +
           tiny(dt), name + "dbank")
    return loss, dq, dbank


def loss_inputs(n, v, d, dt, ignored=0.1, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    bank = torch.nn.functional.normalize(r(v, d), dim=1)
    target = torch.randint(0, v, (n,), generator=gen, device="cuda")
    q = torch.nn.functional.normalize(bank[target] + 0.6 * d ** -0.5 * r(n, d), dim=1)
    target[torch.rand(n, generator=gen, device="cuda") < ignored] = -1
    return q.to(dt), bank.to(dt), target, r(n)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("n,v,d", [(1, 1, 8), (1, 2, 8), (1, 5000, 64), (64, 1024, 256), (128, 256, 64), (129, 257, 72),
                                   (100, 333, 70), (300, 129, 1), (500, 700, 384), (33, 4001, 768), (2000, 3, 16),
                                   (1000, 20000, 128), (257, 1000, 33)])
def test_softmax_loss(n, v, d, dt):
    q, bank, target, g = loss_inputs(n, v, d, dt, seed=n + v + d)
    loss_check(q, bank, target, 1 / 0.07, g)
    loss_check(q, bank, target, 1.0, torch.full_like(g, 1.0 / n))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16])
def test_softmax_loss_in_pieces(dt):
    """n so large that the bank's gradient takes several pieces, the last one shorter and odd."""
    q, bank, target, g = loss_inputs(9000, 10007, 40, dt, seed=4)
    loss_check(q, bank, target, 5.0, g)


@pytest.mark.gpu
def test_softmax_loss_repeated_targets_and_weights():
    q, bank, target, g = loss_inputs(600, 50, 64, F16, ignored=0.0)
    loss_check(q, bank, torch.full_like(target, 17), 8.0, g)
    g[::3] = 0.0
    g[1] = 1e6  # one row far above the others
    loss_check(q, bank, target, 8.0, g)
    loss, dq, dbank = loss_check(q, bank, target, 8.0, torch.zeros_like(g))
    assert not dq.any() and not dbank.any()


@pytest.mark.gpu
def test_softmax_loss_ignored_rows():
    """All rows ignored, and every way of pointing outside the bank; nan in an ignored row stays there."""
    o = ops()
    q, bank, target, g = loss_inputs(200, 300, 48, BF16)
    loss, dq, dbank = loss_check(q, bank, torch.full_like(target, -1), 3.0, g)
    assert not loss.any() and not dq.any() and not dbank.any()
    t = target.clamp(min=0)
    outside = t.clone()
    outside[0], outside[5], outside[9], outside[11] = 300, -100, 2 ** 40, -2 ** 62
    a = loss_check(q, bank, outside, 3.0, g)
    t[[0, 5, 9, 11]] = -1
    b = loss_check(q, bank, t, 3.0, g)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    q2 = q.clone()
    q2[5] = float("nan")
    leaves = [q2.requires_grad_(), bank.clone().requires_grad_()]
    loss, _ = o.softmax_loss(*leaves, t, 3.0)
    dq, dbank = torch.autograd.grad(loss, leaves, g)
    assert torch.equal(loss, b[0]) and torch.equal(dq, b[1])
    assert not dq[5].any()


@pytest.mark.gpu
def test_softmax_loss_large_logits_and_learnt_rows():
    """Logits in the thousands, and rows whose loss is far below the rounding of their lse."""
    q, bank, target, g = loss_inputs(150, 400, 32, BF16, ignored=0.0)
    loss_check((q * 30).to(BF16), (bank * 30).to(BF16), target, 4.0, g)
    eye = torch.eye(64, device="cuda").to(F16)
    t = torch.arange(64, device="cuda")
    loss, _, _ = loss_check(eye, eye, t, 25.0, torch.ones(64, device="cuda"))
    assert torch.allclose(loss.double(), torch.full((64,), math.log1p(63 * math.exp(-25.0)), device="cuda",
                                                    dtype=torch.float64), rtol=1e-5)


@pytest.mark.gpu
def test_softmax_loss_gradient_of_one_leaf_and_views():
    o = ops()
    q, bank, target, g = loss_inputs(130, 500, 64, F16)
    _, dq, dbank = loss_check(q, bank, target, 6.0, g)
    ql = q.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(o.softmax_loss(ql, bank, target, 6.0)[0], ql, g)[0], dq)
    kl = bank.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(o.softmax_loss(q, kl, target, 6.0)[0], kl, g)[0], dbank)
    loss = o.softmax_loss(q, bank, target, 6.0)[0]
    assert torch.equal(o.softmax_loss(q.t().contiguous().t(), bank.t().contiguous().t(), target, 6.0)[0], loss)
    wide = torch.zeros(130 * 2, dtype=torch.int64, device="cuda")
    wide[::2] = target
    assert torch.equal(o.softmax_loss(q, bank, wide[::2], 6.0)[0], loss)
    ql = q.clone().requires_grad_()
    got, = torch.autograd.grad(o.softmax_loss(ql, bank, target, 6.0)[0].sum(), ql)
    want, = torch.autograd.grad(o.softmax_loss(ql, bank, target, 6.0)[0], ql, torch.ones_like(g))
    assert torch.equal(got, want)
    empty = torch.zeros(0, 64, dtype=F16, device="cuda", requires_grad=True)
    none, _ = o.softmax_loss(empty, kl, target[:0], 6.0)
    dk, = torch.autograd.grad(none.sum(), kl)
    assert none.shape == (0,) and not dk.any()


# -- differences, repeatability, graphs, streams, threads -----------------------------------------
@pytest.mark.gpu
def test_gradients_against_differences():
    """Directional derivatives from central differences of the operators' own forward passes.  The
    loss is held in fp32: a step h along a unit direction of bf16-exact size gives the slope to
    (rounding of the loss) / h + h^2 / 6 of the third derivative; both are far below the 2 %."""
    o = ops()
    q, bank, target, g = loss_inputs(40, 90, 32, F16, ignored=0.0, seed=11)
    ql, kl = q.clone().requires_grad_(), bank.clone().requires_grad_()
    f = lambda a, b: (o.softmax_loss(a, b, target, 5.0)[0].double() * g.double()).sum()  # noqa: E731
    dq, dk = torch.autograd.grad(o.softmax_loss(ql, kl, target, 5.0)[0], (ql, kl), g)
    for leaf, grad in ((0, dq), (1, dk)):
        base = (q, bank)[leaf]
        step = (2.0 ** -6 * torch.where(grad >= 0, 1.0, -1.0)).to(F16)
        up, down = (base + step), (base - step)
        moved = (up.double() - down.double())
        diff = (f(up, bank) - f(down, bank)) if leaf == 0 else (f(q, up) - f(q, down))
        want = (grad.double() * moved).sum()
        assert abs(float(diff - want)) <= 0.02 * abs(float(want)), (leaf, float(diff), float(want))


@pytest.mark.gpu
def test_gradients_repeat_bit_for_bit():
    x, w, b, res, g = linear_inputs(30000, 64, 128, F16, res=True)
    q, bank, target, gl = loss_inputs(3000, 9001, 96, BF16)
    xn, wn, bn, gn = norm_inputs(20000, 256, F16, F32)
    o = ops()

    def once():
        lx, lw, lb = (t.detach().clone().requires_grad_() for t in (x, w, b))
        out = list(torch.autograd.grad(o.linear(lx, lw, lb, res, "gelu"), (lx, lw, lb), g))
        lq, lk = (t.detach().clone().requires_grad_() for t in (q, bank))
        out += torch.autograd.grad(o.softmax_loss(lq, lk, target, 9.0)[0], (lq, lk), gl)
        ln = [t.detach().clone().requires_grad_() for t in (xn, wn, bn)]
        return out + list(torch.autograd.grad(o.layer_norm(*ln)[0], ln, gn))

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))
    check_device()


def encoder_block(o, x, p, call_loss, target, scale):
    """One pre-norm feed-forward block, the mean over a window and the loss against its own bank."""
    h = o.layer_norm(x, p["nw"], p["nb"])[0]
    h = o.linear(h, p["w1"], p["b1"], None, "gelu")
    y = o.linear(h, p["w2"], p["b2"], x, "none")
    y = o.layer_norm(y, p["fw"], p["fb"])[0]
    e = torch.nn.functional.normalize(y.float().mean(1), dim=-1).to(x.dtype)
    return call_loss(e, p["bank"], target, scale), e


def block_params(d, f, v, dt, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    p = {"nw": 1 + 0.1 * r(d), "nb": 0.1 * r(d), "w1": r(f, d) * d ** -0.5, "b1": 0.1 * r(f), "w2": r(d, f) * f ** -0.5,
         "b2": 0.1 * r(d), "fw": 1 + 0.1 * r(d), "fb": 0.1 * r(d),
         "bank": torch.nn.functional.normalize(r(v, d), dim=1)}
    return {k: t.to(dt).requires_grad_() for k, t in p.items()}


@pytest.mark.gpu
def test_operators_together_as_an_encoder_block():
    """Norm, feed-forward with residual, norm, window mean and loss, forward and backward, against the
    same chain in 64 bits.  Five roundings to 16 bits lie on the way forward and as many back; with
    random signs they add up to a few u of the norm, and 16 u is the allowance."""
    o, dt = ops(), F16
    p = block_params(64, 256, 500, dt)
    x = torch.randn(24, 50, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dt)
    x.requires_grad_()
    target = torch.arange(24, device="cuda") * 20
    target[3] = -1
    loss, e = encoder_block(o, x, p, lambda *a: o.softmax_loss(*a)[0], target, 10.0)
    leaves = [x] + list(p.values())
    g = torch.full_like(loss, 64.0)
    grads = torch.autograd.grad(loss, leaves, g)
    check_device()

    class Plain:
        @staticmethod
        def layer_norm(x, w, b):
            return (torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, 1e-5),)

        @staticmethod
        def linear(x, w, b, res, act):
            y = x @ w.t() + b
            y = torch.nn.functional.gelu(y) if act == "gelu" else y
            return y if res is None else y + res

    ref = [t.detach().double().requires_grad_() for t in leaves]
    rp = dict(zip(p, ref[1:]))

    def plain_loss(e, bank, t, scale):
        s = scale * e.double() @ bank.t()
        got = torch.logsumexp(s, 1) - s.gather(1, t.clamp(min=0)[:, None])[:, 0]
        return torch.where(t >= 0, got, torch.zeros_like(got))

    h = Plain.layer_norm(ref[0], rp["nw"], rp["nb"])[0]
    h = Plain.linear(h, rp["w1"], rp["b1"], None, "gelu")
    y = Plain.linear(h, rp["w2"], rp["b2"], ref[0], "none")
    y = Plain.layer_norm(y, rp["fw"], rp["fb"])[0]
    want_e = torch.nn.functional.normalize(y.mean(1), dim=-1)
    want = plain_loss(want_e, rp["bank"], target, 10.0)
    want_grads = torch.autograd.grad(want, ref, g.double())
    rel = lambda a, b: float((a.detach().double() - b.detach()).norm() / b.detach().norm())  # noqa: E731
    assert rel(e, want_e.detach()) <= 16 * u(dt)
    assert rel(loss, want.detach()) <= 16 * u(dt)
    for name, a, b in zip(["x"] + list(p), grads, want_grads):
        assert rel(a, b) <= 16 * u(dt), (name, rel(a, b))


@pytest.mark.gpu
def test_captured_training_step_replays_on_new_inputs():
    o, dt = ops(), F16
    p = block_params(64, 128, 300, dt, seed=1)
    x = torch.randn(6, 20, 64, device="cuda").to(dt)
    target = torch.randint(0, 300, (6,), device="cuda")
    leaves = list(p.values())

    def step():
        loss, _ = encoder_block(o, x, p, lambda *a: o.softmax_loss(*a)[0], target, 10.0)
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves, torch.full_like(loss, 64.0)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, each with its own workspaces
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for seed in (1, 2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
        target.copy_(torch.randint(0, 300, (6,), generator=gen, device="cuda"))
        want = step()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    check_device()


@pytest.mark.gpu
def test_capture_beside_a_living_eager_graph():
    """A step is captured while an eager graph of the same leaves waits for its backward pass; both give
    the gradients of a plain step.  (Autograd ties a leaf to the stream that its living graph was made
    on, so the capture takes that stream.)"""
    o, dt = ops(), F16
    p = block_params(64, 128, 300, dt, seed=5)
    x = torch.randn(6, 20, 64, device="cuda").to(dt)
    target = torch.randint(0, 300, (6,), device="cuda")
    leaves = list(p.values())
    forward = lambda: encoder_block(o, x, p, lambda *a: o.softmax_loss(*a)[0], target, 10.0)[0]  # noqa: E731
    backward = lambda loss: torch.autograd.grad(loss, leaves, torch.full_like(loss, 64.0))  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        want = backward(forward())
        waiting = forward()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            got = backward(forward())
        graph.replay()
        late = backward(waiting)
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, late):
        assert torch.equal(a, b) and torch.equal(a, c)
    check_device()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Matrices of more than 2^31 values: rows at both ends equal those of small calls, bit for bit."""
    o = ops()
    gen = torch.Generator(device="cuda").manual_seed(6)
    m, k, n = 2_200_011, 16, 1000
    x = torch.randn((m, k), generator=gen, device="cuda").to(F16)
    w, b = torch.randn((n, k), generator=gen, device="cuda").to(F16), torch.randn(n, generator=gen, device="cuda").to(F16)
    y = o.linear(x, w, b, None, "gelu")
    assert y.numel() > 2 ** 31
    for a in (0, m - 300):
        assert torch.equal(y[a:a + 300], o.linear(x[a:a + 300], w, b, None, "gelu"))
    wn = torch.ones(n, dtype=F16, device="cuda")
    z, mean, rstd = o.layer_norm(y, wn, wn)
    for a in (0, m - 300):
        assert torch.equal(z[a:a + 300], o.layer_norm(y[a:a + 300], wn, wn)[0])
    dx, _, _ = o.layer_norm_backward(z, y, wn, mean, rstd, True, True, True)
    part = slice(m - 300, m)
    assert torch.equal(dx[part], o.layer_norm_backward(z[part], y[part], wn, mean[part], rstd[part], True, False, False)[0])
    del z, dx
    gx, _, _ = o.linear_backward(y, x, w, b, "relu", True, True, True)
    assert torch.equal(gx[part], o.linear_backward(y[part], x[part], w, b, "relu", True, False, False)[0])
    del gx, y, x
    torch.cuda.empty_cache()
    bank = torch.zeros((8_500_003, 256), dtype=BF16, device="cuda")  # all logits 0 but the last row's
    bank[-1, :8] = 1.0
    q = torch.zeros((5, 256), dtype=BF16, device="cuda")
    q[:, 0] = torch.arange(5, device="cuda").to(BF16)
    target = torch.tensor([8_500_002, 8_500_002, 8_500_002, 0, 8_500_002], device="cuda")
    loss, lse = o.softmax_loss(q, bank, target, 1.0)
    want = torch.log(torch.exp(torch.arange(5.0, dtype=torch.float64)) + 8_500_002)
    assert torch.allclose(lse.double().cpu(), want, rtol=1e-6)
    assert torch.allclose(loss.double().cpu(), want - torch.tensor([0.0, 1.0, 2.0, 0.0, 4.0], dtype=torch.float64), rtol=1e-6)
    dq, dbank = o.softmax_loss_backward(torch.ones(5, device="cuda"), q, bank, target, loss, lse, 1.0, True, True)
    p = torch.exp(torch.arange(5.0, dtype=torch.float64) - want)  # of the last row
    for d in range(8):
        assert torch.allclose(dq[[0, 1, 2, 4], d].double().cpu(), (p - 1)[[0, 1, 2, 4]], rtol=2 ** -7)
    last = ((p - torch.tensor([1.0, 1.0, 1.0, 0.0, 1.0])) * torch.arange(5.0, dtype=torch.float64)).sum()
    assert abs(float(dbank[-1, 0]) - float(last)) <= 2 ** -7 * abs(float(last))
    check_device()


@pytest.mark.gpu
def test_two_streams_and_two_threads_at_once():
    import threading
    o = ops()
    x, w, b, _, g = linear_inputs(20000, 128, 256, F16)
    q, bank, target, gl = loss_inputs(1500, 8000, 64, F16)

    def both():
        lx, lw, lb = (t.detach().clone().requires_grad_() for t in (x, w, b))
        out = list(torch.autograd.grad(o.linear(lx, lw, lb, None, "gelu"), (lx, lw, lb), g))
        lq, lk = (t.detach().clone().requires_grad_() for t in (q, bank))
        return out + list(torch.autograd.grad(o.softmax_loss(lq, lk, target, 9.0)[0], (lq, lk), gl))

    want = both()
    torch.cuda.synchronize()
    got, failed = {}, []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                got[i] = [both() for _ in range(3)]
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for runs in got.values():
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(run, want))
    check_device()
