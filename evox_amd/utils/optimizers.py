"""Gradient-based optimizers used by the evolution-strategy family.

A small functional API in the spirit of optax (which the reference relies on but which is not
part of this stack): ``opt = adam(lr)``; ``state = opt.init(params)``; ``updates, state =
opt.update(grads, state, params)``; ``params = apply_updates(params, updates)``.  Parameters may
be any tree of tensors.  ``OptaxWrapper`` makes such an optimizer a ``Stateful`` module whose
state lives in the State tree (reference: ``src/evox/utils/common.py:142-153``), and ``ClipUp``
is the PGPE optimizer of Toklu et al. (reference: ``es_variants/pgpe.py:34-64``).
"""
from __future__ import annotations

from typing import Any, Callable, NamedTuple, Optional

import torch

from ..core import tree as _tree
from ..core.module import Stateful
from ..core.state import State
from ..core.struct import dataclass, pytree_field


class GradientTransformation(NamedTuple):
    init: Callable
    update: Callable


def apply_updates(params, updates):
    return _tree.tree_map(lambda p, u: p + u, params, updates)


def sgd(learning_rate: float, momentum: Optional[float] = None) -> GradientTransformation:
    def init(params):
        if momentum is None:
            return {}
        return {"trace": _tree.tree_map(torch.zeros_like, params)}

    def update(grads, state, params=None):
        if momentum is None:
            return _tree.tree_map(lambda g: -learning_rate * g, grads), state
        trace = _tree.tree_map(lambda t, g: momentum * t + g, state["trace"], grads)
        return _tree.tree_map(lambda t: -learning_rate * t, trace), {"trace": trace}

    return GradientTransformation(init, update)


def adam(learning_rate: float, b1: float = 0.9, b2: float = 0.999, eps: float = 1e-8) -> GradientTransformation:
    def init(params):
        first = _tree.tree_leaves(params)[0]
        return {"count": torch.zeros((), dtype=torch.float32, device=first.device),
                "mu": _tree.tree_map(torch.zeros_like, params), "nu": _tree.tree_map(torch.zeros_like, params)}

    def update(grads, state, params=None):
        count = state["count"] + 1
        mu = _tree.tree_map(lambda m, g: b1 * m + (1 - b1) * g, state["mu"], grads)
        nu = _tree.tree_map(lambda v, g: b2 * v + (1 - b2) * g * g, state["nu"], grads)
        c1 = 1 - b1 ** count
        c2 = 1 - b2 ** count
        updates = _tree.tree_map(lambda m, v: -learning_rate * (m / c1) / (torch.sqrt(v / c2) + eps), mu, nu)
        return updates, {"count": count, "mu": mu, "nu": nu}

    return GradientTransformation(init, update)


def rmsprop(learning_rate: float, decay: float = 0.9, eps: float = 1e-8) -> GradientTransformation:
    def init(params):
        return {"nu": _tree.tree_map(torch.zeros_like, params)}

    def update(grads, state, params=None):
        nu = _tree.tree_map(lambda v, g: decay * v + (1 - decay) * g * g, state["nu"], grads)
        return _tree.tree_map(lambda g, v: -learning_rate * g / (torch.sqrt(v) + eps), grads, nu), {"nu": nu}

    return GradientTransformation(init, update)


class AdamW(GradientTransformation):
    """What :func:`adamw` returns: ``init`` and ``update`` like every optimizer here, and

    ``step(grads, state, params) -> (params, state)``  one whole step (on a GPU one launch per 72 leaves; parameters in
                                                       bfloat16 are rounded once);
    ``moments(state, params=None) -> (mu, nu)``        the running averages as trees like ``params``, or flat (leaf after
                                                       leaf, each padded to a multiple of 256) where none are given."""

    step: Callable
    moments: Callable
    separable: bool      # every variable's step depends on its own gradients alone (8-bit moments share a unit among 32)


def adamw(learning_rate: float, b1: float = 0.9, b2: float = 0.999, eps: float = 1e-8, weight_decay: float = 1e-2,
          state_bits: int = 32, mask=None) -> AdamW:
    """Adam with decoupled weight decay, all leaves of a tree in one kernel (``ops.adamw``).

    ``state_bits=8`` keeps both moments in 8 bits (2.06 bytes per parameter instead of 8; see ``ops.adamw`` for the format).
    ``mask``: a tree of truth values like the parameters, or a function that makes one from them; ``weight_decay`` applies
    where it is true (default: everywhere).  Leaves are float32 or bfloat16."""
    if not (learning_rate >= 0 and 0 <= b1 < 1 and 0 <= b2 < 1 and eps >= 0 and weight_decay >= 0):
        raise ValueError("adamw: learning_rate, eps and weight_decay must not be negative, b1 and b2 lie in [0, 1)")
    if state_bits not in (8, 32):
        raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
    from ..ops import adamw as _aw

    def init(params):
        return _aw.adamw_init(_tree.tree_leaves(params), state_bits)

    def run(grads, state, params, updates):
        if params is None:
            raise ValueError("adamw needs the parameters next to the gradients")
        leaves, treedef = _tree.tree_flatten(params)
        g, gdef = _tree.tree_flatten(grads)
        if gdef != treedef:
            raise ValueError(f"adamw: structure mismatch\n  {treedef}\n  {gdef}")
        decay = None
        if mask is not None:
            decay, mdef = _tree.tree_flatten(mask(params) if callable(mask) else mask)
            if mdef != treedef:
                raise ValueError(f"adamw: the mask's structure differs from the parameters'\n  {treedef}\n  {mdef}")
        if (state["mu"].dtype == torch.uint8) != (state_bits == 8):
            raise ValueError(f"adamw: state_bits={state_bits}, but the state was made for another width")
        out, state = _aw.adamw_step(leaves, g, state, learning_rate=learning_rate, b1=b1, b2=b2, eps=eps,
                                    weight_decay=weight_decay, decay=decay, updates=updates)
        return _tree.tree_unflatten(treedef, out), state

    def update(grads, state, params=None):
        return run(grads, state, params, True)

    def step(grads, state, params):
        return run(grads, state, params, False)

    def moments(state, params=None):
        flat = _aw.adamw_moments(state)
        if params is None:
            return flat
        leaves, treedef = _tree.tree_flatten(params)
        if sum(_aw.padded(p.numel()) for p in leaves) != flat[0].numel():
            raise ValueError("adamw: the state does not belong to these parameters")
        trees = []
        for x in flat:
            parts, at = [], 0
            for p in leaves:
                parts.append(x[at:at + p.numel()].view(p.shape))
                at += _aw.padded(p.numel())
            trees.append(_tree.tree_unflatten(treedef, parts))
        return tuple(trees)

    opt = AdamW(init, update)
    opt.step, opt.moments, opt.separable = step, moments, state_bits == 32
    return opt


_BY_NAME = {"adam": adam, "adamw": adamw, "sgd": sgd, "rmsprop": rmsprop}


def by_name(name: str, learning_rate: float) -> GradientTransformation:
    if name not in _BY_NAME:
        raise ValueError(f"Unknown optimizer {name}")
    return _BY_NAME[name](learning_rate=learning_rate)


@dataclass
class OptaxWrapper(Stateful):
    """A functional optimizer as a module: its state is the ``opt_state`` field of its State."""

    optimizer: Any = pytree_field(static=True)
    init_params: Any = None

    def setup(self, key):
        return State(opt_state=self.optimizer.init(self.init_params))

    def update(self, state, grads, params=None):
        updates, opt_state = self.optimizer.update(grads, state.opt_state, params)
        return updates, state.replace(opt_state=opt_state)

    def step(self, state, grads, params):
        """Parameters after the update: the optimizer's own whole step where it has one (and no subclass its own update)."""
        fused = getattr(self.optimizer, "step", None) if type(self).update is OptaxWrapper.update else None
        if fused is None:
            updates, state = self.update(state, grads, params)
            return apply_updates(params, updates), state
        params, opt_state = fused(grads, state.opt_state, params)
        return params, state.replace(opt_state=opt_state)


def tree_l2_norm(tree):
    return torch.sqrt(sum((leaf ** 2).sum() for leaf in _tree.tree_leaves(tree)))


@dataclass
class ClipUp(Stateful):
    """Normalised-gradient momentum with a velocity norm cap."""

    step_size: float
    max_speed: float
    momentum: float
    params: Any = None

    def setup(self, key):
        return State(velocity=_tree.tree_map(torch.zeros_like, self.params))

    def update(self, state, gradient, _params=None):
        gnorm = tree_l2_norm(gradient)
        velocity = _tree.tree_map(lambda v, g: self.momentum * v + self.step_size * g / gnorm, state.velocity, gradient)
        vnorm = tree_l2_norm(velocity)
        scale = torch.where(vnorm > self.max_speed, self.max_speed / vnorm, torch.ones_like(vnorm))
        velocity = _tree.tree_map(lambda v: v * scale, velocity)
        return _tree.tree_map(lambda v: -v, velocity), state.replace(velocity=velocity)
