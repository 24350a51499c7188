"""``torch.ops.rbq.*``: PyTorch operators over the C ABI of librbq.so.

The reference exposes its CUDA code to Python as JIT-compiled torch extensions
(src/neurosamble/kernels/ops.py:23-68); this path's operators are registered the same way a
torch user finds them, ``torch.ops.rbq.<name>``, each a thin wrapper of one ``rbq_*`` entry
point of include/rbq.h:

  search(h, q, k, nprobe, rerank, prune, probe_split, seeded, query_bits=4)
                                             -> (dist [n, k] f32, ids [n, k] i64)
  rotate(h, x)                               -> xr [n, Dp]                         (rbq_rotate)
  query_prep(h, qr, bits=4)                  -> (planes [n, bits, Dp/32] i32, delta [n], k1 [n])
  coarse(h, qr, nprobe, margin)              -> (probes [n, nprobe] i32, g [n, nprobe] f32)
  scan(h, qr, planes, delta, k1, probes, g, R, prune, slices, cand_cap, tau0)
                                             -> (cand_ids [n, R] i64, cand_dist [n, R] f32)
  bound_seed(h, qr, planes, delta, k1, probes, g, R, cand_cap) -> tau [n] f32
  rerank(h, q, cand_ids, k)                  -> (dist [n, k] f32, ids [n, k] i64)
  merge_results(dist [p, n, k], ids [p, n, k]) -> (dist [n, k], ids [n, k])

and, without an index, the operators of the encoder that makes the vectors, differentiable:

  linear(x [..., k], w [n, k], bias=None, residual=None, act="none") -> y [..., n]   (rbq_linear)
  layer_norm(x [..., d], w [d], b [d], eps=1e-5) -> (y, mean [...], rstd [...])      (rbq_layer_norm)
  softmax_loss(q [n, d], bank [v, d], target [n] i64, scale) -> (loss [n], lse [n])  (rbq_softmax_loss)

linear is act(x w^T + bias) + residual with act "none", "relu" or "gelu" (the erf form); linear and
softmax_loss take float16 or bfloat16, layer_norm also float32, with w and b of x's type or
float32.  A row of softmax_loss whose target lies outside [0, v) is ignored: loss 0, no
gradient.  mean, rstd and lse carry no gradient; the backward passes (linear_backward,
layer_norm_backward, softmax_loss_backward) are operators too and are not differentiable again.

``h`` is the index handle as an int (``IndexIVFRaBitQ.handle.value``).  ``query_bits`` of search
is the search mode: 4 (QUANT4), 8 (QUANT8), 16 (LUT16) or 32 (LUT32); ``bits`` of query_prep is
the query code width, 4 or 8, and scan and bound_seed take it from the planes' shape (the stage
operators cover the two popcount modes).  Inputs are CUDA tensors
on the index's device (made contiguous here); outputs are allocated by PyTorch on that device,
and the work is enqueued on ``torch.cuda.current_stream()`` of it, without synchronising.
Distances are squared L2, ascending; missing results have id -1 and distance +inf.  A failed
call raises RuntimeError with the library's message.  Every operator has a fake
implementation, so output shapes propagate under FakeTensorMode and meta tensors.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.library import custom_op

from . import _lib

Pair = Tuple[Tensor, Tensor]


def _p(t: Optional[Tensor]) -> Optional[ctypes.c_void_p]:
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _st(t: Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _h(handle: int) -> ctypes.c_void_p:
    if not handle:
        raise RuntimeError("rbq: null index handle")
    return ctypes.c_void_p(handle)


def _cuda(t: Tensor, dtype: torch.dtype, name: str) -> Tensor:
    if not t.is_cuda:
        raise RuntimeError(f"rbq: {name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise RuntimeError(f"rbq: {name} must be {dtype}, got {t.dtype}")
    return t.contiguous()


def _dp(d: int) -> int:
    return (d + 31) // 32 * 32


@custom_op("rbq::search", mutates_args=())
def search(handle: int, q: Tensor, k: int, nprobe: int, rerank: int, prune: bool, probe_split: int,
           seeded: int, query_bits: int = 4) -> Pair:
    q = _cuda(q, torch.float32, "q")
    n = q.shape[0]
    sp = _lib.SearchParams()
    _lib.lib().rbq_search_params_default(ctypes.byref(sp))
    sp.n_probes, sp.k, sp.rerank, sp.prune = nprobe, k, rerank, int(prune)
    sp.probe_split, sp.seeded, sp.query_bits = probe_split, seeded, query_bits
    dist = torch.empty((n, k), dtype=torch.float32, device=q.device)
    ids = torch.empty((n, k), dtype=torch.int64, device=q.device)
    with torch.cuda.device(q.device):
        _lib.call("rbq_search", _h(handle), ctypes.byref(sp), _p(q), n, _p(dist), _p(ids), _st(q))
    return dist, ids


@search.register_fake
def _(handle, q, k, nprobe, rerank, prune, probe_split, seeded, query_bits=4):
    n = q.shape[0]
    return q.new_empty((n, k)), q.new_empty((n, k), dtype=torch.int64)


@custom_op("rbq::rotate", mutates_args=())
def rotate(handle: int, x: Tensor) -> Tensor:
    x = _cuda(x, torch.float32, "x")
    out = torch.empty((x.shape[0], _dp(x.shape[1])), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.call("rbq_rotate", _h(handle), _p(x), x.shape[0], _p(out), _st(x))
    return out


@rotate.register_fake
def _(handle, x):
    return x.new_empty((x.shape[0], _dp(x.shape[1])))


def _bits(bits: int) -> int:
    if bits not in (4, 8):
        raise RuntimeError(f"rbq: query bits must be 4 (QUANT4) or 8 (QUANT8), got {bits}")
    return bits


@custom_op("rbq::query_prep", mutates_args=())
def query_prep(handle: int, qr: Tensor, bits: int = 4) -> Tuple[Tensor, Tensor, Tensor]:
    qr = _cuda(qr, torch.float32, "qr")
    n, dp = qr.shape
    planes = torch.empty((n, _bits(bits), dp // 32), dtype=torch.int32, device=qr.device)
    delta = torch.empty(n, dtype=torch.float32, device=qr.device)
    k1 = torch.empty(n, dtype=torch.float32, device=qr.device)
    with torch.cuda.device(qr.device):
        _lib.call("rbq_query_prep", _h(handle), _p(qr), n, _p(planes), _p(delta), _p(k1), bits, _st(qr))
    return planes, delta, k1


@query_prep.register_fake
def _(handle, qr, bits=4):
    n, dp = qr.shape
    return qr.new_empty((n, _bits(bits), dp // 32), dtype=torch.int32), qr.new_empty(n), qr.new_empty(n)


@custom_op("rbq::coarse", mutates_args=())
def coarse(handle: int, qr: Tensor, nprobe: int, margin: int) -> Pair:
    qr = _cuda(qr, torch.float32, "qr")
    n = qr.shape[0]
    probes = torch.empty((n, nprobe), dtype=torch.int32, device=qr.device)
    g = torch.empty((n, nprobe), dtype=torch.float32, device=qr.device)
    with torch.cuda.device(qr.device):
        _lib.call("rbq_coarse", _h(handle), _p(qr), n, nprobe, margin, _p(probes), _p(g), _st(qr))
    return probes, g


@coarse.register_fake
def _(handle, qr, nprobe, margin):
    n = qr.shape[0]
    return qr.new_empty((n, nprobe), dtype=torch.int32), qr.new_empty((n, nprobe))


def _scan_inputs(qr, planes, delta, k1, probes, g):
    return (_cuda(qr, torch.float32, "qr"), _cuda(planes, torch.int32, "planes"),
            _cuda(delta, torch.float32, "delta"), _cuda(k1, torch.float32, "k1"),
            _cuda(probes, torch.int32, "probes"), _cuda(g, torch.float32, "g"))


@custom_op("rbq::scan", mutates_args=())
def scan(handle: int, qr: Tensor, planes: Tensor, delta: Tensor, k1: Tensor, probes: Tensor, g: Tensor, R: int,
         prune: bool, slices: int, cand_cap: int, tau0: Optional[Tensor]) -> Pair:
    qr, planes, delta, k1, probes, g = _scan_inputs(qr, planes, delta, k1, probes, g)
    n, nprobe = probes.shape
    if tau0 is not None:
        tau0 = _cuda(tau0, torch.float32, "tau0")
    ids = torch.empty((n, R), dtype=torch.int64, device=qr.device)
    dist = torch.empty((n, R), dtype=torch.float32, device=qr.device)
    with torch.cuda.device(qr.device):
        _lib.call("rbq_scan", _h(handle), _p(qr), _p(planes), _p(delta), _p(k1), n, _p(probes), _p(g), nprobe,
                  nprobe, _p(tau0), None, None, R, int(prune), slices, cand_cap, _p(ids), _p(dist), None,
                  _bits(planes.shape[1]), _st(qr))
    return ids, dist


@scan.register_fake
def _(handle, qr, planes, delta, k1, probes, g, R, prune, slices, cand_cap, tau0):
    n = probes.shape[0]
    return qr.new_empty((n, R), dtype=torch.int64), qr.new_empty((n, R))


@custom_op("rbq::bound_seed", mutates_args=())
def bound_seed(handle: int, qr: Tensor, planes: Tensor, delta: Tensor, k1: Tensor, probes: Tensor, g: Tensor,
               R: int, cand_cap: int) -> Tensor:
    qr, planes, delta, k1, probes, g = _scan_inputs(qr, planes, delta, k1, probes, g)
    n, nprobe = probes.shape
    tau = torch.empty(n, dtype=torch.float32, device=qr.device)
    with torch.cuda.device(qr.device):
        _lib.call("rbq_bound_seed", _h(handle), _p(qr), _p(planes), _p(delta), _p(k1), n, _p(probes), _p(g),
                  nprobe, nprobe, R, cand_cap, _p(tau), _bits(planes.shape[1]), _st(qr))
    return tau


@bound_seed.register_fake
def _(handle, qr, planes, delta, k1, probes, g, R, cand_cap):
    return qr.new_empty(probes.shape[0])


@custom_op("rbq::rerank", mutates_args=())
def rerank(handle: int, q: Tensor, cand_ids: Tensor, k: int) -> Pair:
    q = _cuda(q, torch.float32, "q")
    cand_ids = _cuda(cand_ids, torch.int64, "cand_ids")
    n, R = cand_ids.shape
    dist = torch.empty((n, k), dtype=torch.float32, device=q.device)
    ids = torch.empty((n, k), dtype=torch.int64, device=q.device)
    with torch.cuda.device(q.device):
        _lib.call("rbq_rerank", _h(handle), _p(q), n, _p(cand_ids), R, k, _p(dist), _p(ids), _st(q))
    return dist, ids


@rerank.register_fake
def _(handle, q, cand_ids, k):
    n = cand_ids.shape[0]
    return q.new_empty((n, k)), q.new_empty((n, k), dtype=torch.int64)


@custom_op("rbq::merge_results", mutates_args=())
def merge_results(dist: Tensor, ids: Tensor) -> Pair:
    dist = _cuda(dist, torch.float32, "dist")
    ids = _cuda(ids, torch.int64, "ids")
    if dist.dim() != 3 or dist.shape != ids.shape:
        raise RuntimeError("rbq: merge_results takes [parts, n, k] distances and ids of one shape")
    p, n, k = dist.shape
    od = torch.empty((n, k), dtype=torch.float32, device=dist.device)
    oi = torch.empty((n, k), dtype=torch.int64, device=dist.device)
    with torch.cuda.device(dist.device):
        _lib.call("rbq_merge_results", _p(dist), _p(ids), p, n, k, _p(od), _p(oi), _st(dist))
    return od, oi


@merge_results.register_fake
def _(dist, ids):
    _, n, k = dist.shape
    return dist.new_empty((n, k)), ids.new_empty((n, k))


# -- operators of the read encoder ---------------------------------------------------------------
_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # RBQ_F16, RBQ_BF16, RBQ_F32
_HALVES = (torch.float16, torch.bfloat16)


def _operand(t: Tensor, like: Tensor, name: str) -> Tensor:
    """t, on like's device and of its type, dense and on a 16-byte boundary."""
    if t.device != like.device or not t.is_cuda:
        raise RuntimeError(f"rbq: {name} must be a CUDA tensor on {like.device}, got {t.device}")
    if t.dtype != like.dtype:
        raise RuntimeError(f"rbq: {name} must be {like.dtype}, got {t.dtype}")
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _first(t: Tensor, types, name: str) -> Tensor:
    if not t.is_cuda:
        raise RuntimeError(f"rbq: {name} must be a CUDA tensor")
    if t.dtype not in types:
        raise RuntimeError(f"rbq: {name} must be {' or '.join(str(x) for x in types)}, got {t.dtype}")
    return _operand(t, t, name)


def _shape(t: Tensor, want, name: str) -> None:
    if tuple(t.shape) != tuple(want):
        raise RuntimeError(f"rbq: {name} must have shape {tuple(want)}, got {tuple(t.shape)}")


def _workspace(device: torch.device, query: str, *args) -> Tuple[Optional[Tensor], int]:
    need = ctypes.c_int64()
    _lib.call(query, *args, ctypes.byref(need))
    if need.value == 0:
        return None, 0
    return torch.empty(need.value, dtype=torch.uint8, device=device), need.value


def _linear_args(x: Tensor, w: Tensor, bias: Optional[Tensor], act: str):
    x = _first(x, _HALVES, "x")
    w = _operand(w, x, "w")
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise RuntimeError(f"rbq: linear takes x [..., k] and w [n, k], got {tuple(x.shape)} and {tuple(w.shape)}")
    if bias is not None:
        bias = _operand(bias, x, "bias")
        _shape(bias, w.shape[:1], "bias")
    if act not in _lib.ACTIVATIONS:
        raise RuntimeError(f"rbq: act must be one of {', '.join(_lib.ACTIVATIONS)}, got {act!r}")
    n, k = w.shape
    if n < 1 or k < 1:
        raise RuntimeError("rbq: linear needs k >= 1 and n >= 1")
    return x, w, bias, x.numel() // k, k, n


@custom_op("rbq::linear", mutates_args=())
def linear(x: Tensor, w: Tensor, bias: Optional[Tensor] = None, residual: Optional[Tensor] = None,
           act: str = "none") -> Tensor:
    x, w, bias, m, k, n = _linear_args(x, w, bias, act)
    out = x.shape[:-1] + (n,)
    if residual is not None:
        residual = _operand(residual, x, "residual")
        _shape(residual, out, "residual")
    y = torch.empty(out, dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        a = _lib.ACTIVATIONS[act]
        ws, size = _workspace(x.device, "rbq_linear_workspace", m, k, n, _TYPES[x.dtype], a, 0)
        _lib.call("rbq_linear", _p(x), _p(w), _p(bias), _p(residual), _p(y), m, k, n, _TYPES[x.dtype], a, _p(ws), size,
                  _st(x))
    return y


@linear.register_fake
def _(x, w, bias=None, residual=None, act="none"):
    return x.new_empty(x.shape[:-1] + (w.shape[0],))


@custom_op("rbq::linear_backward", mutates_args=())
def linear_backward(g: Tensor, x: Tensor, w: Tensor, bias: Optional[Tensor], act: str, need_x: bool, need_w: bool,
                    need_bias: bool) -> Tuple[Tensor, Tensor, Tensor]:
    x, w, bias, m, k, n = _linear_args(x, w, bias, act)
    _shape(g, x.shape[:-1] + (n,), "g")
    g = _operand(g, x, "g")
    dx = torch.empty_like(x) if need_x else x.new_empty(0)
    dw = torch.empty_like(w) if need_w else x.new_empty(0)
    db = x.new_empty(n if need_bias else 0)
    with torch.cuda.device(x.device):
        a = _lib.ACTIVATIONS[act]
        ws, size = _workspace(x.device, "rbq_linear_workspace", m, k, n, _TYPES[x.dtype], a, 1)
        _lib.call("rbq_linear_backward", _p(g), _p(x), _p(w), _p(bias), _p(dx if need_x else None),
                  _p(dw if need_w else None), _p(db if need_bias else None), m, k, n, _TYPES[x.dtype], a, _p(ws), size,
                  _st(x))
    return dx, dw, db


@linear_backward.register_fake
def _(g, x, w, bias, act, need_x, need_w, need_bias):
    return (torch.empty_like(x) if need_x else x.new_empty(0), torch.empty_like(w) if need_w else x.new_empty(0),
            x.new_empty(w.shape[0] if need_bias else 0))


def _linear_context(ctx, inputs, output):
    x, w, bias, _, ctx.act = inputs
    ctx.save_for_backward(x, w, bias)


def _linear_gradient(ctx, g):
    x, w, bias = ctx.saved_tensors
    need = ctx.needs_input_grad + (False,) * 3  # trailing arguments left at their defaults are not listed
    dx = dw = db = None
    if need[0] or need[1] or need[2]:
        dx, dw, db = linear_backward(g, x, w, bias, ctx.act, need[0], need[1], need[2])
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, g if need[3] else None, None)


linear.register_autograd(_linear_gradient, setup_context=_linear_context)


def _norm_args(x: Tensor, w: Tensor):
    x = _first(x, tuple(_TYPES), "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"rbq: layer_norm takes x [..., d] with d >= 1, got {tuple(x.shape)}")
    if w.dtype not in (x.dtype, torch.float32):
        raise RuntimeError(f"rbq: w must be {x.dtype} or torch.float32, got {w.dtype}")
    if w.device != x.device:
        raise RuntimeError(f"rbq: w must be a CUDA tensor on {x.device}, got {w.device}")
    w = w.contiguous()
    d = x.shape[-1]
    _shape(w, (d,), "w")
    return x, w, x.numel() // d, d


@custom_op("rbq::layer_norm", mutates_args=())
def layer_norm(x: Tensor, w: Tensor, b: Tensor, eps: float = 1e-5) -> Tuple[Tensor, Tensor, Tensor]:
    x, w, rows, d = _norm_args(x, w)
    b = _operand(b, w, "b")
    _shape(b, (d,), "b")
    y = torch.empty_like(x)
    mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    with torch.cuda.device(x.device):
        _lib.call("rbq_layer_norm", _p(x), _p(w), _p(b), _p(y), _p(mean), _p(rstd), rows, d, eps, _TYPES[x.dtype],
                  _TYPES[w.dtype], _st(x))
    return y, mean, rstd


@layer_norm.register_fake
def _(x, w, b, eps=1e-5):
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    return torch.empty_like(x), mean, torch.empty_like(mean)


@custom_op("rbq::layer_norm_backward", mutates_args=())
def layer_norm_backward(g: Tensor, x: Tensor, w: Tensor, mean: Tensor, rstd: Tensor, need_x: bool, need_w: bool,
                        need_b: bool) -> Tuple[Tensor, Tensor, Tensor]:
    x, w, rows, d = _norm_args(x, w)
    _shape(g, x.shape, "g")
    g = _operand(g, x, "g")
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        _shape(t, x.shape[:-1], name)
    mean, rstd = _cuda(mean, torch.float32, "mean"), _cuda(rstd, torch.float32, "rstd")
    dx = torch.empty_like(x) if need_x else x.new_empty(0)
    dw, db = w.new_empty(d if need_w else 0), w.new_empty(d if need_b else 0)
    with torch.cuda.device(x.device):
        ws, size = (_workspace(x.device, "rbq_layer_norm_backward_workspace", rows, d) if need_w or need_b
                    else (None, 0))
        _lib.call("rbq_layer_norm_backward", _p(g), _p(x), _p(w), _p(mean), _p(rstd), _p(dx if need_x else None),
                  _p(dw if need_w else None), _p(db if need_b else None), rows, d, _TYPES[x.dtype], _TYPES[w.dtype],
                  _p(ws), size, _st(x))
    return dx, dw, db


@layer_norm_backward.register_fake
def _(g, x, w, mean, rstd, need_x, need_w, need_b):
    d = x.shape[-1]
    return (torch.empty_like(x) if need_x else x.new_empty(0), w.new_empty(d if need_w else 0),
            w.new_empty(d if need_b else 0))


def _norm_context(ctx, inputs, output):
    x, w, _, _ = inputs
    _, mean, rstd = output
    ctx.mark_non_differentiable(mean, rstd)
    ctx.save_for_backward(x, w, mean, rstd)


def _norm_gradient(ctx, g, _mean, _rstd):
    x, w, mean, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dw, db = layer_norm_backward(g, x, w, mean, rstd, need[0], need[1], need[2])
    return dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None


layer_norm.register_autograd(_norm_gradient, setup_context=_norm_context)


def _loss_args(q: Tensor, bank: Tensor, target: Tensor):
    q = _first(q, _HALVES, "q")
    bank = _operand(bank, q, "bank")
    if q.dim() != 2 or bank.dim() != 2 or q.shape[1] != bank.shape[1] or bank.shape[0] < 1 or q.shape[1] < 1:
        raise RuntimeError(f"rbq: softmax_loss takes q [n, d] and bank [v, d] with v, d >= 1, got {tuple(q.shape)} and "
                           f"{tuple(bank.shape)}")
    target = _cuda(target, torch.int64, "target")
    if target.device != q.device:
        raise RuntimeError(f"rbq: target must be a CUDA tensor on {q.device}, got {target.device}")
    _shape(target, q.shape[:1], "target")
    return q, bank, target


@custom_op("rbq::softmax_loss", mutates_args=())
def softmax_loss(q: Tensor, bank: Tensor, target: Tensor, scale: float) -> Pair:
    q, bank, target = _loss_args(q, bank, target)
    (n, d), v = q.shape, bank.shape[0]
    loss = torch.empty(n, dtype=torch.float32, device=q.device)
    lse = torch.empty_like(loss)
    with torch.cuda.device(q.device):
        ws, size = _workspace(q.device, "rbq_softmax_loss_workspace", n, v, d, _TYPES[q.dtype], 0)
        _lib.call("rbq_softmax_loss", _p(q), _p(bank), _p(target), n, v, d, scale, _TYPES[q.dtype], _p(loss), _p(lse),
                  _p(ws), size, _st(q))
    return loss, lse


@softmax_loss.register_fake
def _(q, bank, target, scale):
    loss = q.new_empty(q.shape[0], dtype=torch.float32)
    return loss, torch.empty_like(loss)


@custom_op("rbq::softmax_loss_backward", mutates_args=())
def softmax_loss_backward(g: Tensor, q: Tensor, bank: Tensor, target: Tensor, loss: Tensor, lse: Tensor, scale: float,
                          need_q: bool, need_bank: bool) -> Pair:
    q, bank, target = _loss_args(q, bank, target)
    (n, d), v = q.shape, bank.shape[0]
    for t, name in ((g, "g"), (loss, "loss"), (lse, "lse")):
        _shape(t, (n,), name)
    g, loss, lse = (_cuda(t, torch.float32, name) for t, name in ((g, "g"), (loss, "loss"), (lse, "lse")))
    dq = torch.empty_like(q) if need_q else q.new_empty(0)
    dbank = torch.empty_like(bank) if need_bank else q.new_empty(0)
    with torch.cuda.device(q.device):
        ws, size = _workspace(q.device, "rbq_softmax_loss_workspace", n, v, d, _TYPES[q.dtype], 1)
        _lib.call("rbq_softmax_loss_backward", _p(g), _p(q), _p(bank), _p(target), _p(loss), _p(lse), n, v, d, scale,
                  _TYPES[q.dtype], _p(dq if need_q else None), _p(dbank if need_bank else None), _p(ws), size, _st(q))
    return dq, dbank


@softmax_loss_backward.register_fake
def _(g, q, bank, target, loss, lse, scale, need_q, need_bank):
    return (torch.empty_like(q) if need_q else q.new_empty(0), torch.empty_like(bank) if need_bank else q.new_empty(0))


def _loss_context(ctx, inputs, output):
    q, bank, target, ctx.scale = inputs
    loss, lse = output
    ctx.mark_non_differentiable(lse)
    ctx.save_for_backward(q, bank, target, loss, lse)


def _loss_gradient(ctx, g, _lse):
    q, bank, target, loss, lse = ctx.saved_tensors
    need = ctx.needs_input_grad
    dq, dbank = softmax_loss_backward(g, q, bank, target, loss, lse, ctx.scale, need[0], need[1])
    return dq if need[0] else None, dbank if need[1] else None, None, None


softmax_loss.register_autograd(_loss_gradient, setup_context=_loss_context)
