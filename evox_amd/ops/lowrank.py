"""Populations of low-rank changes of a shared layer (kernels: ``csrc/lowrank*.hip``).

Individual p of a population differs from a shared linear layer by a product of rank r, ``W + s A_pᵀ B_p``, and, where
the layer has own biases, by ``s c_p``.  Evaluating it takes one product with the shared weights for all rows and
``2 r (in + out)`` operations per row, where a population of full matrices takes one matrix per individual from memory; the
evolution-strategy gradient of the shared weights is ``Σ_p w_p A_pᵀ B_p``, one product over all individuals' factors.

``lowrank_linear``        the layer on rows of all individuals, or on rows (requests) that name their individual
``lowrank_weighted_sum``  the fitness-weighted sum of all individuals' changes
"""
from __future__ import annotations

import ctypes
from numbers import Real

import torch

from .. import _native
from ._util import DTYPE_CODE, check, hip, launch_device, on_gpu, stream_of

P, I, I64, F = _native.P, _native.I, _native.I64, _native.F
_native.register_hip_api({
    "evox_hip_lowrank_linear_ws": (I64, [P, P, P, P, P, P, P, P, P]),
    "evox_hip_lowrank_linear_kernel": (I, [P, P, P, P, P, P, P, P, P]),
    "evox_hip_lowrank_linear": (I, [P, P, P, P, P, P, P, P, P, P, I64, F, P]),
    "evox_hip_lowrank_sum_ws": (I64, [P, P, P, P, P, P, P]),
    "evox_hip_lowrank_sum_kernel": (I, [P, P, P, P, P, P, P]),
    "evox_hip_lowrank_sum": (I, [P, P, P, P, P, P, P, P, I64, F, P]),
})

_ACT = {"identity": 0, "tanh": 1, "relu": 2, "sigmoid": 3}
_ACT_FN = {"identity": lambda v: v, "tanh": torch.tanh, "relu": torch.relu, "sigmoid": torch.sigmoid}
_INDEX = {torch.int32: 1, torch.int64: 2}
_MOST = 2 ** 31 - 2 ** 16          # features are indexed in 32 bits, up to the end of the last tile


def _check_factors(what, a, b):
    sa, sb = a.shape, b.shape
    for name, shape in (("a", sa), ("b", sb)):
        if len(shape) != 3:
            raise ValueError(f"{what}: {name} has three dimensions (individuals, rank, features), got shape {tuple(shape)}")
    if a.dtype not in DTYPE_CODE or b.dtype not in DTYPE_CODE:
        raise TypeError(f"{what} takes float32 or bfloat16 factors, got {a.dtype} and {b.dtype}")
    r = sa[1]
    if sb[0] != sa[0] or not r <= sb[1] <= r + 1 or r < 1:
        raise ValueError(f"{what}: a is (P, r, in) and b (P, r, out) or, with own biases, (P, r + 1, out), r >= 1; got "
                         f"{tuple(sa)} and {tuple(sb)}")
    if a.dtype is not b.dtype:
        raise TypeError(f"{what}: the factors have different types, {a.dtype} and {b.dtype}")
    if sa[2] < 1:
        raise ValueError(f"{what} needs at least one input feature")
    if r >= _MOST or sa[2] >= _MOST or sb[2] >= _MOST:
        raise ValueError(f"{what}: a factor's rank and features lie below 2^31 - 2^16")
    return r, sb[1] - r


def _no_grad_wanted(what, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} builds no autograd graph: detach its inputs, or call it under torch.no_grad()")


def _packed(t):
    """Factors with each individual's rows contiguous (individuals at any stride)."""
    return t if t.stride(2) == 1 and (t.stride(1) == t.shape[2] or t.shape[1] == 1) else t.contiguous()


def lowrank_linear(x: torch.Tensor, weight: torch.Tensor, a: torch.Tensor, b: torch.Tensor, index=None, bias=None,
                   scale: float = 1.0, activation: str = "identity") -> torch.Tensor:
    """``act(x W + bias + scale · ((x A_pᵀ) B_p + c_p))``.

    weight : (in, out) shared by all individuals
    a, b   : (P, r, in) and (P, r, out) factors; a further row of b, (P, r + 1, out), is the individual's own bias c_p
    x      : (P, E, in) or (P, in), rows of individual p in x[p] — or, with ``index`` (T,) int32 / int64, (T, in), row t by
             individual ``index[t]``; an index outside [0, P) takes the shared part alone (no factors are read for it)
    bias   : (out,) or None;  activation: identity, tanh, relu or sigmoid
    →        x's leading dimensions with out in the place of in, in x's type, contiguous

    ``x``, ``weight``, ``a``, ``b`` are all float32 or all bfloat16; sums are float32 and the result is rounded once.  ``x`` may be
    strided or expanded over individuals, the factors may be views of wider rows (``MLP.lowrank_factors``).  No autograd graph
    is built: inputs that ask for a gradient are refused, and so is a y of 2^24 tiles or more, which are 64 x 64 at least (2^30 rows of up
    to 64 outputs)."""
    r, own_bias = _check_factors("lowrank_linear", a, b)
    if weight.dim() != 2 or weight.shape[0] != a.shape[2] or weight.shape[1] != b.shape[2]:
        raise ValueError(f"lowrank_linear: a weight of shape {tuple(weight.shape)} does not fit factors of {a.shape[2]} inputs and "
                         f"{b.shape[2]} outputs")
    if x.dtype != a.dtype or weight.dtype != a.dtype:
        raise TypeError(f"lowrank_linear: x, weight and factors have one type, got {x.dtype}, {weight.dtype} and {a.dtype}")
    n_in, n_out, pop = weight.shape[0], weight.shape[1], a.shape[0]
    if index is None:
        if x.dim() not in (2, 3) or x.shape[0] != pop or x.shape[-1] != n_in:
            raise ValueError(f"lowrank_linear: x is ({pop}, rows, {n_in}) or ({pop}, {n_in}), got {tuple(x.shape)}")
    else:
        if x.dim() != 2 or x.shape[1] != n_in:
            raise ValueError(f"lowrank_linear: with an index, x is (rows, {n_in}), got {tuple(x.shape)}")
        if index.dtype not in _INDEX:
            raise TypeError(f"lowrank_linear: the index is int32 or int64, got {index.dtype}")
        if tuple(index.shape) != (x.shape[0],):
            raise ValueError(f"lowrank_linear: {x.shape[0]} rows but an index of shape {tuple(index.shape)}")
    if bias is not None:
        if tuple(bias.shape) != (n_out,):
            raise ValueError(f"lowrank_linear: the bias has shape ({n_out},), got {tuple(bias.shape)}")
        if bias.dtype not in DTYPE_CODE:
            raise TypeError(f"lowrank_linear: the bias is float32 or bfloat16, got {bias.dtype}")
    if not isinstance(scale, Real):
        raise TypeError("lowrank_linear: scale is a number")
    if activation not in _ACT:
        raise ValueError(f"lowrank_linear: activation is one of {sorted(_ACT)}, got {activation!r}")
    _no_grad_wanted("lowrank_linear", x, weight, a, b, bias)
    dev = x.device
    where = x.get_device()
    for t in (weight, a, b, index, bias):
        if t is not None and t.get_device() != where:
            raise ValueError("lowrank_linear: inputs on different devices")
    if not on_gpu(x):
        return lowrank_linear_reference(x, weight, a, b, index, bias, scale, activation)
    y = x.new_empty((*x.shape[:-1], n_out))
    if y.numel() == 0:
        return y
    if x.stride(-1) != 1 and n_in > 1:
        x = x.contiguous()
    rows = y.numel() // n_out
    per = x.shape[1] if x.dim() == 3 else 1
    weight = weight.contiguous()
    a, b = _packed(a), _packed(b)
    bias = bias if bias is None else bias.to(torch.float32).contiguous()
    index = index if index is None else index.contiguous()
    lib = hip()
    dims = (ctypes.c_int64 * 7)(rows, pop, per, x.stride(0), x.stride(1) if x.dim() == 3 else 0, a.stride(0), b.stride(0))
    ints = (ctypes.c_int * 7)(n_in, n_out, r, own_bias, _ACT[activation], DTYPE_CODE[x.dtype],
                              0 if index is None else _INDEX[index.dtype])
    call = (x.data_ptr(), weight.data_ptr(), a.data_ptr(), b.data_ptr(), None if bias is None else bias.data_ptr(),
            None if index is None else index.data_ptr(), y.data_ptr(), ctypes.addressof(dims), ctypes.addressof(ints))
    floats = lib.evox_hip_lowrank_linear_ws(*call)
    if floats < 0:
        raise ValueError(f"lowrank_linear: {rows} rows of {n_out} outputs are more tiles than one launch holds (2^24 of 64 x 64)")
    ws = x.new_empty(floats, dtype=torch.float32) if floats > 0 else None
    with launch_device(dev):
        check(lib.evox_hip_lowrank_linear(*call, None if ws is None else ws.data_ptr(), floats, float(scale), stream_of(y)), "lowrank_linear")
    return y


def lowrank_linear_reference(x, weight, a, b, index=None, bias=None, scale=1.0, activation="identity"):
    """The layer in float32 tensor operations."""
    r, own_bias = a.shape[1], b.shape[1] > a.shape[1]
    x3 = x.float() if x.dim() == 3 else x.float()[:, None, :]
    a32, b32 = a.float(), b.float()
    if index is not None:
        on = (index >= 0) & (index < a.shape[0])
        at = torch.where(on, index, torch.zeros_like(index)).long()
        if a.shape[0] == 0:
            a32, b32 = a32.new_zeros(1, *a.shape[1:]), b32.new_zeros(1, *b.shape[1:])
        a32, b32 = a32[at], b32[at]
    d = torch.matmul(torch.matmul(x3, a32.transpose(1, 2).contiguous()), b32[:, :r].contiguous())
    if own_bias:
        d = d + b32[:, r:]
    d = d * scale
    if index is not None:
        d = torch.where(on[:, None, None], d, torch.zeros_like(d))
    y = torch.matmul(x3, weight.float()) + d
    if bias is not None:
        y = y + bias.float()
    y = _ACT_FN[activation](y).to(x.dtype)
    return y if x.dim() == 3 else y[:, 0]


def lowrank_weighted_sum(w: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0):
    """``(scale · Σ_p w_p A_pᵀ B_p, scale · Σ_p w_p c_p)``: (in, out) and (out,) in float32, the second None without own biases.

    w : (P,) float32;  a : (P, r, in), b : (P, r, out) or (P, r + 1, out) as in :func:`lowrank_linear`, float32 or bfloat16
    views of any stride between individuals.  Sums are float32 in an order that depends on sizes, strides and alignment alone
    (repeated calls give the same bits).  A factor that is not finite leaves its row or column of the sum not finite, and nothing
    else.  With bfloat16 factors a product w a is held to 24 bits from 2e-31 on (to 2^-126 below) and up to 3.39e38.  No autograd
    graph is built: inputs that ask for a gradient are refused, and so are results of 2^24 tiles of 64 x 64 or more."""
    r, own_bias = _check_factors("lowrank_weighted_sum", a, b)
    pop = a.shape[0]
    if w.dtype != torch.float32:
        raise TypeError(f"lowrank_weighted_sum takes float32 weights, got {w.dtype}")
    if tuple(w.shape) != (pop,):
        raise ValueError(f"lowrank_weighted_sum: {pop} individuals but weights of shape {tuple(w.shape)}")
    if not isinstance(scale, Real):
        raise TypeError("lowrank_weighted_sum: scale is a number")
    _no_grad_wanted("lowrank_weighted_sum", w, a, b)
    dev = w.device
    if a.device != dev or b.device != dev:
        raise ValueError("lowrank_weighted_sum: inputs on different devices")
    if not on_gpu(w):
        return lowrank_weighted_sum_reference(w, a, b, scale)
    n_in, n_out = a.shape[2], b.shape[2]
    g = w.new_empty((n_in, n_out))
    gb = w.new_empty(n_out) if own_bias else None
    if n_out == 0:
        return g, gb
    if pop == 0:
        return g.zero_(), gb if gb is None else gb.zero_()
    w, a, b = w.contiguous(), _packed(a), _packed(b)
    lib = hip()
    dims = (ctypes.c_int64 * 3)(pop, a.stride(0), b.stride(0))
    ints = (ctypes.c_int * 4)(n_in, n_out, r, DTYPE_CODE[a.dtype])
    call = (w.data_ptr(), a.data_ptr(), b.data_ptr(), g.data_ptr(), None if gb is None else gb.data_ptr(), ctypes.addressof(dims),
            ctypes.addressof(ints))
    floats = lib.evox_hip_lowrank_sum_ws(*call)
    if floats < 0:
        raise ValueError(f"lowrank_weighted_sum: {n_in} x {n_out} results are more tiles than one launch holds (2^24 of 64 x 64)")
    ws = w.new_empty(floats) if floats > 0 else None
    with launch_device(dev):
        check(lib.evox_hip_lowrank_sum(*call, None if ws is None else ws.data_ptr(), floats, float(scale), stream_of(g)), "lowrank_weighted_sum")
    return g, gb


def lowrank_weighted_sum_reference(w, a, b, scale=1.0):
    """The sums in float32 tensor operations."""
    r = a.shape[1]
    wa = (a.float() * w[:, None, None]).flatten(0, 1)
    b32 = b.float()
    g = scale * (wa.T @ b32[:, :r].flatten(0, 1))
    return g, (scale * (w @ b32[:, r]) if b.shape[1] > r else None)
