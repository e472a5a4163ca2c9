"""Measured cases of the low-rank population operators and of the fused AdamW step.

``lowrank_linear``        every individual (or request) has its own rank-r change of a shared layer:
                          y = act(x W + bias + scale ((x A_p^T) B_p + c_p))
``lowrank_weighted_sum``  the layer's share of an evolution-strategy gradient: G = sum_p w_p A_p^T B_p, g = sum_p w_p c_p
``adamw``                 one AdamW step of all leaves of a parameter tree, moments in 32 or in 8 bits

``run`` computes them in elementary torch operations, or, where ``own`` is true, through ``evox_amd``.
"""
import math

import torch

own = False

DEVICE = "cuda"
F32, BF16 = "float32", "bfloat16"
ALIGN = 256                                # every leaf's moments start at a multiple of this many elements
BLOCK = 32                                 # 8-bit moments that share one power-of-two scale
LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.999, 1e-8, 1e-2
ACTIVATIONS = {"identity": lambda v: v, "tanh": torch.tanh, "relu": torch.relu, "sigmoid": torch.sigmoid}


def _policy(*sizes):
    return ",".join("%dx%d,%d" % (i, o, o) for i, o in zip(sizes[:-1], sizes[1:]))


def listed():
    return [
        # one environment step of 4096 small locomotion policies: launch latency
        dict(name="linear hopper", op="linear", pop=4096, per=1, inp=32, out=32, rank=1, dtype=F32, act="tanh", own_bias=True, index=False),
        # the widest layer of the million-parameter policy, one observation per individual
        dict(name="linear 1m policy", op="linear", pop=4096, per=1, inp=1024, out=720, rank=4, dtype=BF16, act="tanh", own_bias=True, index=False),
        # a handful of requests for different individuals of a trained population, some for the centre itself
        dict(name="linear requests", op="linear", pop=300, per=5, inp=4096, out=4096, rank=16, dtype=BF16, act="identity", own_bias=False, index=True),
        # supervised fitness in fp32: 256 individuals on 64 samples each
        dict(name="linear dataset fp32", op="linear", pop=256, per=64, inp=1024, out=1024, rank=8, dtype=F32, act="relu", own_bias=True, index=False),
        # supervised fitness of a large layer: 256 individuals on 256 samples each
        dict(name="linear dataset", op="linear", pop=256, per=256, inp=2048, out=2048, rank=16, dtype=BF16, act="relu", own_bias=True, index=False),
        # gradient of the first layer of the hopper policy, large population
        dict(name="sum hopper", op="sum", pop=16384, inp=11, out=32, rank=1, dtype=F32, own_bias=True),
        # gradient of the widest layer of the million-parameter policy
        dict(name="sum 1m policy", op="sum", pop=4096, inp=1024, out=720, rank=4, dtype=BF16, own_bias=True),
        # gradient of a large layer at the highest rank in use
        dict(name="sum large", op="sum", pop=4096, inp=2048, out=2048, rank=16, dtype=BF16, own_bias=False),
        # the hopper policy's six leaves: launch latency
        dict(name="adamw hopper", op="adamw", leaves=_policy(11, 32, 32, 3), bits=32, param=F32, grad=F32),
        # 67 M parameters in bf16 with fp32 gradients and moments
        dict(name="adamw 67m", op="adamw", leaves=_policy(2048, 8192, 4097, 4096), bits=32, param=BF16, grad=F32),
        # the million-parameter policy (its leaves end inside a block of 32)
        dict(name="adamw8 1m policy", op="adamw", leaves=_policy(244, 1024, 720, 17), bits=8, param=F32, grad=F32),
        # 134 M fp32 parameters with moments in 8 bits
        dict(name="adamw8 134m", op="adamw", leaves=_policy(4096, 16384, 4096, 33), bits=8, param=F32, grad=F32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "sum", "adamw", "adamw"])
    if op == "adamw":
        total, n = _log(rng, 1000, 100_000_000), rng.randint(1, 6)
        sizes = [_log(rng, 1, max(2, int(math.sqrt(total / n)))) for _ in range(n)]
        sizes = [max(1, min(16384, int(math.sqrt(total / n)))) if k == 0 else s for k, s in enumerate(sizes)]
        sizes.append(max(1, min(16384, total // n // sizes[-1])))
        bits = rng.choice([32, 8])
        return dict(op=op, leaves=_policy(*sizes), bits=bits, param=rng.choice([F32, BF16]), grad=rng.choice([F32, BF16]))
    inp, out = _log(rng, 3, 4096), _log(rng, 1, 4096)
    rank, dtype = _log(rng, 1, 16), rng.choice([F32, BF16])
    pop = _log(rng, 16, 16384)
    most = 2.0 ** 39 if dtype == BF16 else 2.0 ** 35          # flops of a drawn case (the listed ones cost more)
    while pop * rank * (inp + out) > 2 ** 29:
        pop = max(1, pop // 2)
    if op == "sum":
        while 2.0 * pop * rank * inp * out > most:
            pop = max(1, pop // 2)
        return dict(op=op, pop=pop, inp=inp, out=out, rank=rank, dtype=dtype, own_bias=rng.random() < 0.5)
    index = rng.random() < 0.4
    per = _log(rng, 1, 4096) if index else _log(rng, 1, 300)  # with an index: the number of requests
    rows = per if index else pop * per
    while rows > 1 and (2.0 * rows * inp * out > most or rows * (inp + out) > 2 ** 28):
        per = max(1, per // 2)
        pop = pop if index else max(1, pop // 2)
        rows = per if index else pop * per
    return dict(op=op, pop=pop, per=per, inp=inp, out=out, rank=rank, dtype=dtype, act=rng.choice(list(ACTIVATIONS)),
                own_bias=rng.random() < 0.5, index=index)


def _shapes(case):
    return [tuple(int(d) for d in s.split("x")) for s in case["leaves"].split(",")]


def _padded(shape):
    return -(-math.prod(shape) // ALIGN) * ALIGN


def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        per = 2 * (4 if case["param"] == F32 else 2) + (4 if case["grad"] == F32 else 2)
        # moments: read and written; 8-bit ones also come back as the bf16 values they stand for
        per += 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4
        return {"bytes": n * per, "flops": 15.0 * n}
    size = 4 if case["dtype"] == F32 else 2
    inp, out, r, extra = case["inp"], case["out"], case["rank"], int(case["own_bias"])
    if case["op"] == "sum":
        p = case["pop"]
        return {"bytes": p * (r * inp + (r + extra) * out) * size + 4 * p + 4 * (inp + extra) * out,
                "flops": 2.0 * p * r * inp * out + 2.0 * p * extra * out}
    rows = case["per"] if case["index"] else case["pop"] * case["per"]
    used = min(rows, case["pop"])
    return {"bytes": (rows * (inp + out) + inp * out + used * (r * inp + (r + extra) * out)) * size + 4 * out + (8 * rows if case["index"] else 0),
            "flops": 2.0 * rows * (inp * out + r * (inp + out))}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=DEVICE).to(dtype)

    if case["op"] == "adamw":
        return _prepare_adamw(case, gen, normal)
    dt = getattr(torch, case["dtype"])
    p, inp, out, r, extra = case["pop"], case["inp"], case["out"], case["rank"], int(case["own_bias"])
    # the factors of one layer lie in one row per individual: [A (r x in), B (r x out), c (out)]
    width = r * inp + (r + extra) * out
    factors = normal(p, -(-width // 8) * 8, dtype=dt)
    s = dict(case=case, a=factors[:, :r * inp].unflatten(1, (r, inp)), b=factors[:, r * inp:width].unflatten(1, (r + extra, out)))
    if case["op"] == "sum":
        s["w"] = normal(p)                                    # centred fitness
        s["scale"] = 1.0 / (p * 0.05)
        return s
    rows = case["per"] if case["index"] else p * case["per"]
    s["weight"] = (normal(inp, out) / math.sqrt(inp)).to(dt)
    s["bias"] = 0.1 * normal(out)
    s["scale"] = 0.05 / math.sqrt(r)
    x = normal(rows, inp, dtype=dt)
    s["x"] = x if case["index"] else x.view(p, case["per"], inp)
    # requests: any individual, about one in eight for the centre alone (-1)
    s["index"] = None
    if case["index"]:
        idx = torch.randint(0, p, (rows,), generator=gen, device=DEVICE)
        s["index"] = torch.where(torch.rand(rows, generator=gen, device=DEVICE) < 0.125, -1, idx)
        s["index"][rows // 2] = -1
    return s


def _prepare_adamw(case, gen, normal):
    shapes = _shapes(case)
    pdt, gdt = getattr(torch, case["param"]), getattr(torch, case["grad"])
    params = [normal(*s).mul_(0.05).to(pdt) for s in shapes]
    grads = [normal(*s).mul_(1e-2).to(gdt) for s in shapes]
    total = sum(_padded(s) for s in shapes)
    inside = torch.zeros(total, dtype=torch.bool, device=DEVICE)
    at = 0
    for s in shapes:
        inside[at:at + math.prod(s)] = True
        at += _padded(s)
    count = torch.tensor(41.0, device=DEVICE)
    if case["bits"] == 32:
        mu = normal(total).mul_(3e-3) * inside
        nu = normal(total).square_().mul_(4e-6) * inside
        return dict(case=case, params=params, grads=grads, state={"count": count, "mu": mu, "nu": nu})
    def codes(lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=gen, device=DEVICE, dtype=torch.uint8)
    # codes of the upper range, as states that have taken some steps hold them: mu about 1e-3, nu about 1e-6
    mu = (codes(70, 127, total) | (codes(0, 2, total) << 7)) * inside
    nu = codes(130, 255, total) * inside
    state = {"count": count, "mu": mu, "nu": nu, "mu_scale": codes(98, 102, total // BLOCK), "nu_scale": codes(71, 75, total // BLOCK)}
    return dict(case=case, params=params, grads=grads, state=state)


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    return {"linear": _plain_linear, "sum": _plain_sum, "adamw": _plain_adamw}[op](state)


def _own(s, op):
    if op == "linear":
        from evox_amd.ops.lowrank import lowrank_linear

        return lowrank_linear(s["x"], s["weight"], s["a"], s["b"], index=s["index"], bias=s["bias"], scale=s["scale"],
                              activation=s["case"]["act"])
    if op == "sum":
        from evox_amd.ops.lowrank import lowrank_weighted_sum

        return lowrank_weighted_sum(s["w"], s["a"], s["b"], scale=s["scale"])
    from evox_amd.utils import optimizers

    opt = optimizers.adamw(LR, b1=B1, b2=B2, eps=EPS, weight_decay=WD, state_bits=s["case"]["bits"])
    params, state = opt.step(s["grads"], s["state"], s["params"])
    mu, nu = opt.moments(state)
    return {"params": params, "count": state["count"], "mu": mu, "nu": nu}


# ------------------------------------------------------------------ plain forms

def _plain_linear(s):
    case, x, w = s["case"], s["x"].float(), s["weight"].float()
    r = case["rank"]
    a, b = s["a"].float(), s["b"].float()
    if s["index"] is None:
        t = x @ a.transpose(1, 2).contiguous()                                     # (P, E, r)
        d = t @ b[:, :r].contiguous()
        if case["own_bias"]:
            d = d + b[:, r:]
    else:
        idx = s["index"].clamp(0, case["pop"] - 1)
        t = (x[:, None, :] * a[idx]).sum(-1)
        d = (t[:, :, None] * b[idx][:, :r]).sum(1)
        if case["own_bias"]:
            d = d + b[idx][:, r]
        d = torch.where((s["index"] >= 0)[:, None], d, torch.zeros_like(d))
    y = (x.reshape(-1, case["inp"]) @ w).view(*x.shape[:-1], case["out"]) + s["bias"] + s["scale"] * d
    return ACTIVATIONS[case["act"]](y).to(s["x"].dtype)


def _plain_sum(s):
    r, inp, out = s["case"]["rank"], s["case"]["inp"], s["case"]["out"]
    w = s["w"] * s["scale"]
    a = (s["a"].float() * w[:, None, None]).reshape(-1, inp)
    b = s["b"].float()
    g = a.T @ b[:, :r].reshape(-1, out)
    return g, (w @ b[:, r] if s["case"]["own_bias"] else None)


def _dither(count, n):
    """(u_mu, u_nu), each (n,) in [0, 1): element i at step t takes the fractional parts of i phi + t (alpha_1, alpha_2), in 32-bit
    fixed point."""
    i = torch.arange(n, device=DEVICE, dtype=torch.int64) * 0x9E3779B9
    t = count.to(torch.int64)
    return tuple((((i + t * c) & 0xFFFFFFFF) >> 16).float() * 2.0 ** -16 for c in (0x91E10DA5, 0xC13FA9A9))


def _pow2(e):
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _decode(code, scale, signed):
    """Codes to values: sign, 4 exponent and 3 mantissa bits where `signed`, else 5 and 3; the lowest exponent holds 0 to 7 units."""
    c = code.to(torch.int64) & (0x7F if signed else 0xFF)
    e, m = c >> 3, c & 7
    v = torch.where(e > 0, (m + 8) << (e - 1).clamp(min=0), m).float()
    if signed:
        v = torch.where(code > 127, -v, v)
    return v * _pow2(scale.to(torch.int32) - 127).repeat_interleave(BLOCK)


def _requantised(v, u, signed):
    """The values that 8-bit codes of v stand for: blocks of 32 share the smallest power-of-two unit whose largest code holds the
    block's largest magnitude; magnitudes are rounded down or up by the dither u, a positive second moment never to zero."""
    bits = 14 if signed else 30
    big = v.abs().view(-1, BLOCK).amax(1)
    unit = ((big.view(torch.int32) >> 23) - 127 - 3 - bits).clamp(min=-126)
    unit = unit + (big > 14.0 * 2.0 ** bits * _pow2(unit)).int()
    y = v.abs() * _pow2(-unit).repeat_interleave(BLOCK)
    shift = ((y.view(torch.int32) >> 23) - 127).clamp(min=3) - 3
    n = torch.floor(y * _pow2(-shift) + u)
    if not signed:
        n = torch.where((n == 0) & (v > 0), torch.ones_like(n), n)
    q = n * _pow2(shift) * _pow2(unit).repeat_interleave(BLOCK)
    return torch.where(v < 0, -q, q).to(torch.bfloat16)


def _flat(leaves):
    pads = [_padded(t.shape) - t.numel() for t in leaves]
    return torch.cat([torch.nn.functional.pad(t.float().reshape(-1), (0, k)) for t, k in zip(leaves, pads)])


def _plain_adamw(s):
    state, leaves, bits = s["state"], s["params"], s["case"]["bits"]
    p, g = _flat(leaves), _flat(s["grads"])
    count = state["count"] + 1
    c1, c2 = ((1 - b ** count.double()).float() for b in (B1, B2))
    mu, nu = state["mu"], state["nu"]
    if bits == 8:
        mu, nu = _decode(mu, state["mu_scale"], True), _decode(nu, state["nu_scale"], False)
    mu = B1 * mu + (1 - B1) * g
    nu = B2 * nu + (1 - B2) * g * g
    new = p - LR * ((mu / c1) / (torch.sqrt(nu / c2) + EPS) + WD * p)
    if bits == 8:
        u_mu, u_nu = _dither(count, mu.numel())
        mu, nu = _requantised(mu, u_mu, True), _requantised(nu, u_nu, False)
    parts = new.split([_padded(t.shape) for t in leaves])
    return {"params": [v[:t.numel()].view(t.shape).to(t.dtype) for v, t in zip(parts, leaves)], "count": count, "mu": mu, "nu": nu}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    r = case["rank"]
    a, b = s["a"].double(), s["b"].double()
    if case["op"] == "sum":
        w = s["w"].double() * s["scale"]
        g = torch.zeros(case["inp"], case["out"], dtype=torch.float64, device=DEVICE)
        for j in range(r):
            g.addmm_((a[:, j] * w[:, None]).T.contiguous(), b[:, j].contiguous())
        return g, ((b[:, r] * w[:, None]).sum(0) if case["own_bias"] else None)
    act = {"identity": lambda v: v, "tanh": lambda v: 1 - 2 / (torch.exp(2 * v) + 1), "relu": lambda v: v.clamp(min=0),
           "sigmoid": lambda v: 1 / (1 + torch.exp(-v))}[case["act"]]
    x = s["x"].double()
    y = torch.matmul(x.reshape(-1, case["inp"]), s["weight"].double()).view(*x.shape[:-1], case["out"])
    y += s["bias"].double()
    used = s["index"] if s["index"] is not None else torch.arange(case["pop"], device=DEVICE)
    at = used.clamp(min=0)
    on = (used >= 0).double() * s["scale"]
    on = on[:, None] if s["index"] is not None else on[:, None, None]
    for j in range(r):
        aj, bj = a[:, j][at], b[:, j][at]
        if s["index"] is None:
            y += on * (x * aj[:, None]).sum(-1, keepdim=True) * bj[:, None]
        else:
            y += on * (x * aj).sum(-1, keepdim=True) * bj
    if case["own_bias"]:
        c = b[:, r][at]
        y += on * (c[:, None] if s["index"] is None else c)
    return act(y)


def _exact_values(code, scale, signed):
    """code -> value by a table of all 256 codes."""
    table = []
    for c in range(256):
        e, m = divmod(c & 127 if signed else c, 8)
        v = float(m) if e == 0 else float(m + 8) * 2.0 ** (e - 1)
        table.append(-v if signed and c >= 128 else v)
    values = torch.tensor(table, dtype=torch.float64, device=DEVICE)[code.long()]
    return (values.view(-1, BLOCK) * torch.pow(2.0, scale.double() - 127)[:, None]).view(-1)


def _exact_rounded(v, step_constant, count, signed):
    blocks = v.view(-1, BLOCK)
    big = blocks.abs().amax(1, keepdim=True)
    top = 14 * 2.0 ** (14 if signed else 30)
    unit = torch.pow(2.0, torch.ceil(torch.log2(big / top)).clamp(min=-126.0))
    y = blocks.abs() / unit
    step = torch.pow(2.0, torch.frexp(y)[1].double() - 4).clamp(min=1.0)
    phase = torch.arange(v.numel(), device=DEVICE).mul_(0x9E3779B9).add_(count * step_constant)
    u = torch.remainder(phase, 2 ** 32).div_(2 ** 16, rounding_mode="floor").double().div_(2.0 ** 16)
    n = torch.floor(y / step + u.view(-1, BLOCK))
    if not signed:
        n = torch.where(blocks > 0, n.clamp(min=1.0), n)
    return (torch.sign(blocks) * n * step * unit).view(-1)


def _exact_adamw(s):
    state, bits = s["state"], s["case"]["bits"]
    t = int(state["count"].item()) + 1
    if bits == 32:
        mu, nu = state["mu"].double(), state["nu"].double()
    else:
        mu, nu = _exact_values(state["mu"], state["mu_scale"], True), _exact_values(state["nu"], state["nu_scale"], False)
    params, at = [], 0
    for p, g in zip(s["params"], s["grads"]):
        n = p.numel()
        g64, p64 = g.double().reshape(-1), p.double().reshape(-1)
        mu[at:at + n].mul_(B1).add_(g64, alpha=1 - B1)
        nu[at:at + n].mul_(B2).addcmul_(g64, g64, value=1 - B2)
        step = (mu[at:at + n] / (1 - B1 ** t)) / (torch.sqrt(nu[at:at + n] / (1 - B2 ** t)) + EPS) + WD * p64
        params.append((p64 - LR * step).view(p.shape))
        at += _padded(p.shape)
    if bits == 8:
        mu, nu = _exact_rounded(mu, 0x91E10DA5, t, True), _exact_rounded(nu, 0xC13FA9A9, t, False)
    return {"params": params, "count": float(t), "mu": mu, "nu": nu}
