"""AdamW over many tensors at once, moments in 32 or in 8 bits (kernel: ``csrc/adamw.hip``).

The moments of all leaves live in one flat buffer each: leaf after leaf in the order given, every leaf padded with zeros
to a multiple of ``ALIGN`` elements.  A state is a dict of tensors:

``count``                  float32 scalar, steps taken (stays at 2^24, and the dither of 8-bit moments stands still from there on)
``mu``, ``nu``             ``(total,)`` float32, or uint8 codes
``mu_scale``, ``nu_scale`` (8 bits only) ``(total / BLOCK,)`` uint8: ``BLOCK`` neighbours share the unit ``2^(scale - 127)``

Codes: ``mu`` sign, 4 exponent and 3 mantissa bits, ``nu`` 5 exponent and 3 mantissa bits; exponent e > 0 and mantissa m stand
for ``(8 + m) 2^(e - 1)`` units, e = 0 for ``m`` units, ``0x7f`` / ``0xff`` for NaN (an infinite moment becomes NaN).  A
block's unit is the smallest that holds its largest magnitude; magnitudes are rounded down or up by a dither that is
equidistributed over the steps, so slow averages move as they should (rounding to nearest would freeze them)."""
from __future__ import annotations

import ctypes
import math
from typing import List, Sequence

import torch

from .. import _native
from ._util import DTYPE_CODE, check, hip, launch_device, stream_of

ALIGN = 256
BLOCK = 32
_MOST = (2 ** 32 - 1) // 256 * 1024               # elements of a leaf on a GPU: 1024 a workgroup, whose threads are counted in 32 bits
_PHASE, _STEP_MU, _STEP_NU = 0x9E3779B9, 0x91E10DA5, 0xC13FA9A9

P, I, I64 = _native.P, _native.I, _native.I64
_native.register_hip_api({
    "evox_hip_adamw": (I, [I, I, P, P, P, P, P, P, I, P, P, P, P, P, P, P, P, P, P, I64, P]),
    "evox_hip_adamw_read": (I, [P, P, P, P, P, P, I64, P]),
})


def padded(n: int) -> int:
    """Elements that a leaf of ``n`` takes in the flat moments."""
    return -(-n // ALIGN) * ALIGN


def adamw_init(params: Sequence[torch.Tensor], state_bits: int = 32) -> dict:
    """The state before the first step."""
    _check_leaves(params, "params")
    if state_bits not in (8, 32):
        raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
    dev = params[0].device
    total = sum(padded(p.numel()) for p in params)
    state = {"count": torch.zeros((), dtype=torch.float32, device=dev)}
    if state_bits == 32:
        state["mu"] = torch.zeros(total, dtype=torch.float32, device=dev)
        state["nu"] = torch.zeros(total, dtype=torch.float32, device=dev)
    else:
        for name in ("mu", "nu"):
            state[name] = torch.zeros(total, dtype=torch.uint8, device=dev)
            state[name + "_scale"] = torch.ones(total // BLOCK, dtype=torch.uint8, device=dev)
    return state


def _check_leaves(leaves, what):
    if not leaves:
        raise ValueError(f"adamw needs at least one tensor in {what}")
    for t in leaves:
        if not isinstance(t, torch.Tensor) or t.dtype not in DTYPE_CODE:
            raise TypeError(f"adamw takes float32 or bfloat16 tensors, got "
                            f"{t.dtype if isinstance(t, torch.Tensor) else type(t).__name__} in {what}")
        if t.get_device() != leaves[0].get_device():
            raise ValueError(f"adamw: the tensors of {what} are on different devices")


def _check_state(state, device, total):
    bits = 8 if state["mu"].dtype is torch.uint8 else 32
    moment = torch.uint8 if bits == 8 else torch.float32
    want = (("count", torch.float32, 1), ("mu", moment, total), ("nu", moment, total))
    if bits == 8:
        want += (("mu_scale", torch.uint8, total // BLOCK), ("nu_scale", torch.uint8, total // BLOCK))
    for name, dtype, n in want:
        t = state.get(name)
        if t is None or t.dtype is not dtype or t.numel() != n or t.device != device or not t.is_contiguous():
            raise ValueError(f"adamw: the state's {name!r} does not belong to these parameters "
                             f"(expected {n} contiguous {dtype} elements on {device})")
    return bits


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], state: dict, *, learning_rate: float,
               b1: float = 0.9, b2: float = 0.999, eps: float = 1e-8, weight_decay: float = 1e-2, decay: Sequence[bool] = None,
               updates: bool = False):
    """One step: ``(new parameters, new state)``, or with ``updates`` the amounts to add in the place of the parameters.

    ``params`` and ``grads`` are lists of float32 or bfloat16 tensors of pairwise equal shapes (any strides; types may differ
    from leaf to leaf and between a parameter and its gradient), ``decay`` says for each leaf whether ``weight_decay`` applies
    to it (default: to all).  Arithmetic is float32 whatever the types, results have the parameters' types and are contiguous.
    Nothing is written in place, no autograd graph is built.  On a GPU all leaves take one launch per 72 of them, and
    a leaf holds fewer than 2^34 elements."""
    if len(params) != len(grads):
        raise ValueError(f"adamw: {len(params)} parameters but {len(grads)} gradients")
    if decay is not None and len(decay) != len(params):
        raise ValueError("adamw: decay needs one entry per parameter")
    if not params:
        raise ValueError("adamw needs at least one tensor in params")
    # one pass over the leaves: a tree of many small ones is bound by it
    total, sizes, flags = 0, [], []
    try:
        where = params[0].get_device()
        for p, g in zip(params, grads):
            flags.append(DTYPE_CODE[p.dtype] | DTYPE_CODE[g.dtype] << 1)
            if p.shape != g.shape:
                raise ValueError(f"adamw: a parameter of shape {tuple(p.shape)} has a gradient of shape {tuple(g.shape)}")
            if p.get_device() != where or g.get_device() != where:
                raise ValueError("adamw: parameters and gradients are on different devices")
            n = p.numel()
            sizes.append(n)
            total += -(-n // ALIGN) * ALIGN
    except (AttributeError, KeyError):
        _check_leaves(params, "params")
        _check_leaves(grads, "grads")
        raise
    if total > _MOST and where >= 0 and max(sizes) > _MOST:
        raise ValueError(f"adamw: a tensor of {max(sizes)} elements is more than one launch holds ({_MOST})")
    device = params[0].device
    bits = _check_state(state, device, total)
    hyper = (learning_rate, b1, b2, 1 - b1, 1 - b2, eps, weight_decay, math.log(b1) if b1 else -math.inf,
             math.log(b2) if b2 else -math.inf)
    if where < 0:
        return adamw_step_reference(params, grads, state, hyper, bits, decay, updates)
    if total == 0:
        return [torch.empty_like(p) for p in params], {**{k: v.clone() for k, v in state.items()}, "count": state["count"] + 1}
    return _step_hip(params, grads, sizes, flags, state, hyper, bits, decay, updates, total, device)


def _step_hip(params, grads, sizes, flags, state, hyper, bits, decay, updates, total, device):
    n = len(params)
    new, out, p_at, g_at, o_at = {}, [], [], [], []
    kept = []                                       # contiguous copies, alive until the launch
    for p, g in zip(params, grads):
        if not p.is_contiguous():
            p = p.contiguous()
            kept.append(p)
        if not g.is_contiguous():
            g = g.contiguous()
            kept.append(g)
        o = torch.empty_like(p)                     # (two microseconds less than naming shape, type and device)
        out.append(o)
        p_at.append(p.data_ptr())
        g_at.append(g.data_ptr())
        o_at.append(o.data_ptr())
    flags = [f | 4 for f in flags] if decay is None else [f | bool(d) << 2 for f, d in zip(flags, decay)]
    new["count"] = torch.empty_like(state["count"])
    new["mu"], new["nu"] = torch.empty_like(state["mu"]), torch.empty_like(state["nu"])
    scales = new_scales = (None, None)
    if bits == 8:
        new["mu_scale"], new["nu_scale"] = torch.empty_like(state["mu_scale"]), torch.empty_like(state["nu_scale"])
        scales = (state["mu_scale"].data_ptr(), state["nu_scale"].data_ptr())
        new_scales = (new["mu_scale"].data_ptr(), new["nu_scale"].data_ptr())
    table = (ctypes.c_int64 * (5 * n))(*p_at, *g_at, *o_at, *sizes, *flags)
    at = ctypes.addressof(table)
    h = (ctypes.c_float * 9)(*hyper)
    with launch_device(device):
        check(hip().evox_hip_adamw(bits, n, at, at + 8 * n, at + 16 * n, at + 24 * n, at + 32 * n, ctypes.addressof(h), int(updates),
                                   state["count"].data_ptr(), new["count"].data_ptr(), state["mu"].data_ptr(),
                                   state["nu"].data_ptr(), *scales, new["mu"].data_ptr(), new["nu"].data_ptr(), *new_scales,
                                   total, stream_of(out[0])), "adamw")
    return out, new


def adamw_moments(state: dict):
    """The flat moments ``(mu, nu)`` that a state holds: float32 as they are, or the bfloat16 values that 8-bit codes stand for
    (exact: a code has four significant bits and its unit is a power of two)."""
    if state["mu"].dtype != torch.uint8:
        return state["mu"], state["nu"]
    names = ("mu", "nu", "mu_scale", "nu_scale")
    total = state["mu"].numel()
    device = state["mu"].device
    if total % ALIGN:
        raise ValueError(f"adamw: moments hold a multiple of {ALIGN} elements, got {total}")
    _check_state(state, device, total)
    if device.type != "cuda":
        return tuple(decode(state[k], state[k + "_scale"], k == "mu").to(torch.bfloat16) for k in ("mu", "nu"))
    mu, nu = (torch.empty_like(state[k], dtype=torch.bfloat16) for k in ("mu", "nu"))
    with launch_device(device):
        check(hip().evox_hip_adamw_read(*(state[k].data_ptr() for k in names), mu.data_ptr(), nu.data_ptr(), total,
                                        stream_of(mu)), "adamw_read")
    return mu, nu


# ------------------------------------------------------------------ the same in tensor operations (host tensors, oracle)

def _pow2(e: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(torch.ones(e.shape, dtype=torch.float32, device=e.device), e)


def decode(codes: torch.Tensor, scale: torch.Tensor, signed: bool) -> torch.Tensor:
    c = codes.to(torch.int64)
    mag = c & 0x7F if signed else c
    e, m = mag >> 3, mag & 7
    v = torch.where(e > 0, (m + 8) << (e - 1).clamp(min=0), m).to(torch.float32)
    v = v * _pow2(scale.to(torch.int32) - 127).repeat_interleave(BLOCK)
    v = torch.where(mag == (0x7F if signed else 0xFF), torch.full_like(v, math.nan), v)
    return torch.where(c > 0x7F, -v, v) if signed else v


def dither(step: int, n: int, constant: int, device=None) -> torch.Tensor:
    phase = torch.arange(n, dtype=torch.int64, device=device) * _PHASE + step * constant
    return ((phase & 0xFFFFFFFF) >> 16).to(torch.float32) * 2.0 ** -16


def encode(v: torch.Tensor, u: torch.Tensor, signed: bool):
    """``(codes, scales)`` of a flat float32 tensor, rounded by the dither ``u``."""
    bits = 14 if signed else 30
    finite = torch.isfinite(v)
    mag = torch.where(finite, v.abs(), torch.zeros_like(v))
    big = mag.view(-1, BLOCK).amax(1)
    unit = ((big.view(torch.int32) >> 23) - 130 - bits).clamp(min=-126)
    unit = unit + (big > 14.0 * 2.0 ** bits * _pow2(unit)).to(torch.int32)
    y = torch.ldexp(mag, -unit.repeat_interleave(BLOCK))
    shift = ((y.view(torch.int32) >> 23) - 127).clamp(min=3) - 3
    code = torch.floor(torch.ldexp(y, -shift) + u).to(torch.int32) + 8 * shift
    if signed:
        code = torch.where(finite, code, torch.full_like(code, 0x7F)) | (torch.signbit(v).to(torch.int32) << 7)
    else:
        code = torch.where((code == 0) & (v > 0), torch.ones_like(code), code)
        code = torch.where(finite, code, torch.full_like(code, 0xFF))
    return code.to(torch.uint8), (unit + 127).to(torch.uint8)


def adamw_step_reference(params, grads, state, hyper, bits, decay=None, updates=False):
    lr, b1, b2, omb1, omb2, eps, wd, _, _ = hyper
    count = state["count"] + 1
    t = float(count)
    c1, c2 = -math.expm1(t * math.log(b1)) if b1 else 1.0, -math.expm1(t * math.log(b2)) if b2 else 1.0
    new = {"count": count}
    if bits == 32:
        mu, nu = state["mu"].clone(), state["nu"].clone()
    else:
        mu, nu = decode(state["mu"], state["mu_scale"], True), decode(state["nu"], state["nu_scale"], False)
    out: List[torch.Tensor] = []
    at = 0
    for k, (p, g) in enumerate(zip(params, grads)):
        n = p.numel()
        p32, g32 = p.detach().reshape(-1).float(), g.detach().reshape(-1).float()
        m, v = mu[at:at + n], nu[at:at + n]
        m.copy_(b1 * m + omb1 * g32)
        v.copy_(b2 * v + omb2 * g32 * g32)
        d = (m / c1) / (torch.sqrt(v / c2) + eps)
        if wd and (decay is None or decay[k]):
            d = d + wd * p32
        out.append((-lr * d if updates else p32 - lr * d).to(p.dtype).reshape(p.shape))
        at += padded(n)
    if bits == 32:
        new["mu"], new["nu"] = mu, nu
    else:
        for name, x, c in (("mu", mu, _STEP_MU), ("nu", nu, _STEP_NU)):
            new[name], new[name + "_scale"] = encode(x, dither(int(t), x.numel(), c, x.device), name == "mu")
    return out, new
