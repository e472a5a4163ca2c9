"""The low-rank kernels where they are large: workspaces, launches, precision, and every variant that a size chooses."""
import ctypes
import math

import pytest
import torch

from evox_amd import _native
from evox_amd._native import build
from evox_amd.core import random as rnd
from evox_amd.models import MLP
from evox_amd.ops.lowrank import lowrank_linear, lowrank_weighted_sum
from test_lowrank import ACT, DEVICES, DTYPES, U, check_linear, check_sum, layer, linear_oracle, randn

needs_library = pytest.mark.skipif(not (build.HIP_LIB.exists() or build.have_hipcc()), reason="no kernel library")


# ------------------------------------------------------------------ what a call asks for, on the host (nothing is launched)

def host_call(dims, ints):
    """The arguments of an entry point up to its sizes, with addresses that are never read."""
    at = 1 << 40
    return at, (ctypes.c_int64 * len(dims))(*dims), (ctypes.c_int * len(ints))(*ints)


def linear_workspace(rows, n_in, n_out, r, dtype=torch.float32, pop=1, per=1):
    at, dims, ints = host_call((rows, pop, per, per * n_in, n_in, r * n_in, r * n_out), (n_in, n_out, r, 0, 0, int(dtype == torch.bfloat16), 0))
    return _native.hip().evox_hip_lowrank_linear_ws(at, at, at, at, None, None, at, ctypes.addressof(dims), ctypes.addressof(ints))


def sum_workspace(pop, n_in, n_out, r, dtype=torch.float32):
    at, dims, ints = host_call((pop, r * n_in, r * n_out), (n_in, n_out, r, int(dtype == torch.bfloat16)))
    return _native.hip().evox_hip_lowrank_sum_ws(at, at, at, at, None, ctypes.addressof(dims), ctypes.addressof(ints))


@needs_library
@pytest.mark.parametrize("dtype", DTYPES)
def test_workspace_of_wide_rows(dtype):
    """Rows of 2^31 bytes and more that are copied to aligned ones have room for their copies."""
    size = torch.finfo(dtype).bits // 8
    for n in (2 ** 31 // size - 5, 2 ** 31 // size + 1, 2 ** 30 + 1):
        assert linear_workspace(17, n, 1024, 1, dtype, pop=17) >= 17 * n * size // 4
        assert sum_workspace(64, n, 256, 1, dtype) >= 64 * n * size // 4
        assert sum_workspace(64, 256, n, 1, dtype) >= 64 * n * size // 4


@needs_library
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_sums_are_divided(dtype):
    """A workgroup counts its terms in 32 bits: sums of more than 2^31 terms are divided (each part has its partial sums) even where
    the outputs alone fill the chip."""
    for pop in (2 ** 31, 2 ** 31 + 17, 2 ** 33):
        assert sum_workspace(pop, 8192, 8192, 1, dtype) >= pop // 2 ** 30 * 8193 * 8192
    assert sum_workspace(2 ** 30, 8192, 8192, 1, dtype) == 0


@needs_library
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_of_very_many_inputs(dtype):
    """Up to four rows take a workgroup for each 128 inputs and 512 threads each: from 2^30 inputs on that is more than a launch counts,
    and they take the tiles that divide the inputs into fewer parts."""
    for n_out, few, many in ((8, 2 ** 29, 2 ** 30), (1024, 2 ** 26, 2 ** 29)):
        assert kernel_of(dtype, 1, 4, few, n_out, 2) == FEW
        assert kernel_of(dtype, 1, 4, many, n_out, 2) == 16


@needs_library
@pytest.mark.parametrize("dtype", DTYPES)
def test_divided_inputs_near_2_to_31(dtype):
    """The parts of K are counted without passing 2^31: tiles of 16 and 64 rows and those of any size have room for all their parts."""
    n = 2 ** 31 - 2 ** 17
    for rows, n_out, kernel, parts in ((4, 8, 16, 512), (100, 8, 64, 256), (5, 7, 0, 256)):
        assert kernel_of(dtype, rows, 1, n, n_out, 1) == kernel
        assert linear_workspace(rows, n, n_out, 1, dtype, pop=rows) >= parts * rows * n_out


def test_refuses_features_near_2_to_31():
    """Tiles are counted in 32 bits beyond a tensor's last feature."""
    n = 2 ** 31 - 2 ** 16
    one = torch.zeros(1, 1, 1)
    wide, weight = one.expand(1, 1, n), torch.zeros(1, 1).expand(n, 1)
    with pytest.raises(ValueError, match="2\\^31"):
        lowrank_linear(wide, weight, wide, one)
    with pytest.raises(ValueError, match="2\\^31"):
        lowrank_linear(one, weight.t(), one, wide)
    with pytest.raises(ValueError, match="2\\^31"):
        lowrank_weighted_sum(torch.zeros(1), wide, one)


@pytest.mark.gpu
def test_copied_rows_beyond_2_to_31_bytes(cuda):
    """17 rows (one, expanded) of 2^30 + 1 bf16 inputs, copied to aligned rows of 2 GiB each; all but a few inputs are zero."""
    n = 2 ** 30 + 1
    at = torch.tensor([0, 1, 7, 8, 2 ** 29 + 3, 2 ** 30 - 1, 2 ** 30], device=cuda)
    gen = torch.Generator().manual_seed(29)
    few = [randn(gen, 1, 7, dtype=torch.bfloat16).to(cuda), randn(gen, 7, 8, dtype=torch.bfloat16).to(cuda), randn(gen, 1, 1, 7, dtype=torch.bfloat16).to(cuda)]
    x, weight, a = (torch.zeros(s, dtype=torch.bfloat16, device=cuda) for s in ((1, n), (n, 8), (1, 1, n)))
    x[:, at], weight[at], a[:, :, at] = few
    b = randn(gen, 1, 1, 8, dtype=torch.bfloat16).to(cuda)
    y = lowrank_linear(x.expand(17, n), weight, a.expand(17, 1, n), b.expand(17, 1, 8))
    check_linear(y, few[0].expand(17, 7), few[1], few[2].expand(17, 1, 7), b.expand(17, 1, 8))


# ------------------------------------------------------------------ launches

@pytest.mark.gpu
@pytest.mark.parametrize("grouped", [True, False])
def test_more_rows_than_threads_of_one_launch(cuda, grouped):
    """16.8 M rows of rank 16 (all of them one individual's 256, expanded): sixty-four lanes for each four of a row's entries of t
    are more threads than a launch counts."""
    gen = torch.Generator().manual_seed(31)
    n_in, n_out, r, per, pop = 264, 72, 16, 256, 65537
    weight, a, b = layer(gen, 1, n_in, n_out, r, 1, torch.bfloat16, cuda)
    x = randn(gen, 1, per, n_in, dtype=torch.bfloat16).to(cuda)
    if grouped:
        want = lowrank_linear(x, weight, a, b, activation="tanh")
        y = lowrank_linear(x.expand(pop, per, n_in), weight, a.expand(pop, -1, -1), b.expand(pop, -1, -1), activation="tanh")
        check_linear(y[-1:], x, weight, a, b, activation="tanh")
        assert torch.equal(y, y[-1:].expand(pop, per, n_out)) and torch.allclose(y[:1].float(), want.float(), atol=0.02)
    else:
        x = x[0, :1].expand(pop * per, n_in)
        index = torch.zeros(pop * per, dtype=torch.int32, device=cuda)
        y = lowrank_linear(x, weight, a, b, index=index, activation="tanh")
        check_linear(y[-3:], x[-3:], weight, a, b, index=index[-3:], activation="tanh")
        assert torch.equal(y, y[-1:].expand(pop * per, n_out))


@needs_library
@pytest.mark.parametrize("dtype", DTYPES)
def test_launches_of_many_rows(dtype):
    """Any number of rows whose tiles fit a launch, whatever their rank; 2^24 tiles and more are refused."""
    for r in (1, 16, 64, 20000):
        assert linear_workspace(2 ** 24, 264, 72, r, dtype, pop=2 ** 16, per=2 ** 8) >= 0
        assert linear_workspace(2 ** 28, 8, 8, r, dtype, pop=2 ** 28) >= 0
        assert linear_workspace(2 ** 30 + 64, 8, 8, r, dtype, pop=2 ** 30 + 64) < 0
        assert sum_workspace(3, 2 ** 29, 5, r, dtype) >= 0
        assert sum_workspace(3, 2 ** 30, 5, r, dtype) < 0 and sum_workspace(3, 5, 2 ** 30 + 1, r, dtype) < 0


# ------------------------------------------------------------------ precision of the weighted sum

PRECISION = [(16384, 136, 130, 1), (4096, 1024, 720, 4), (16384, 512, 520, 1), (20000, 256, 128, 3)]   # individuals, in, out, rank


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", PRECISION, ids=str)
def test_sums_of_few_weights_keep_their_precision(device, dtype, shape):
    """Weights that are zero for all individuals but n (truncation, elites) leave n r terms and their roundings, however long the sum is.

    A term's factors: w a is rounded once and b multiplies it exactly or with one more rounding; each of at most three parts of it is
    added to the running sum, U of that at most whichever way it rounds, and the scale rounds once.  One individual: at most
    3 r + 3 roundings of the terms' magnitudes, entry by entry.  16 individuals: an instruction may round once for each term of
    its step, 24 n times in all; the running sums of signed terms grow with the root of their number, so these errors add up to
    U sqrt(24 n / 6) of the result in norm, and 3 U for the rest."""
    pop, n_in, n_out, r = shape
    gen = torch.Generator().manual_seed(sum(shape))
    _, a, b = layer(gen, pop, n_in, n_out, r, 1, dtype, device)
    for n in (1, 16):
        w = torch.zeros(pop)
        at = torch.randperm(pop, generator=gen)[:n]
        w[at] = randn(gen, n)
        g, gb = lowrank_weighted_sum(w.to(device), a, b, scale=0.7)
        w64, a64, b64 = w[at].double(), a.cpu()[at].double(), b.cpu()[at].double()
        terms = 0.7 * w64[:, None, None, None] * a64[..., None] * b64[:, :r, None, :]
        want, mag = terms.sum((0, 1)), terms.abs().sum((0, 1))
        err = (g.cpu().double() - want).abs()
        if n == 1:
            assert bool((err <= (3 * r + 3) * U * mag).all()), float((err / mag).max() / U)
        else:
            assert float(err.norm()) <= U * (math.sqrt(4 * n) + 3) * float(want.norm()), float(err.norm() / want.norm() / U)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", PRECISION, ids=str)
def test_long_sums_are_as_precise_as_the_tensor_form(cuda, dtype, shape):
    """100 weights and all of them: off by half as much again as one float32 matrix product, and 4 U for the three parts."""
    pop, n_in, n_out, r = shape
    gen = torch.Generator().manual_seed(sum(shape) + 1)
    _, a, b = layer(gen, pop, n_in, n_out, r, 0, dtype, cuda)
    for n in (100, pop):
        w = torch.zeros(pop)
        at = torch.randperm(pop, generator=gen)[:n]
        w[at] = randn(gen, n)
        w = w.to(cuda)
        aw = (a.double() * w.double()[:, None, None]).reshape(-1, n_in)
        want = aw.T.contiguous() @ b.double().reshape(-1, n_out)
        plain = (a.float() * w[:, None, None]).reshape(-1, n_in).T.contiguous() @ b.float().reshape(-1, n_out)
        got, _ = lowrank_weighted_sum(w, a, b)
        err, err_plain = (float((g.double() - want).norm() / want.norm()) for g in (got, plain))
        assert err <= 1.5 * err_plain + 4 * U, (err, err_plain)


# ------------------------------------------------------------------ values at the ends of the range

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per", [1, 16, 40])
def test_infinite_factors(device, dtype, per):
    """Infinite and NaN factors give what the formula gives, an infinity of the right sign among them."""
    gen = torch.Generator().manual_seed(per)
    pop, n_in, n_out, r = 64 // per + 30, 128, 136, 3
    weight, a, b = layer(gen, pop, n_in, n_out, r, 1, dtype, device)
    x = torch.randint(-3, 4, (pop, per, n_in), generator=gen).to(dtype).to(device)   # (t in few bits: nothing is left of it behind 8)
    a.copy_(torch.randint(-2, 3, a.shape, generator=gen))
    b[0, 0, 3], b[1, 2, 70], b[2, 1, 5], b[3, 3, 135] = math.inf, -math.inf, math.nan, math.inf
    a[4, 1, 9], a[5, 0, 127] = math.inf, math.nan
    x[6, 0, 0] = -math.inf
    b[7, 0, :], b[7, 1, :] = math.inf, -math.inf
    y = lowrank_linear(x, weight, a, b, scale=0.5).cpu().double()
    # the own part entry by entry: t_j B_j, so that no product of a matrix library decides what 0 times infinity is
    x64, w64, a64, b64 = x.cpu().double(), weight.cpu().double(), a.cpu().double(), b.cpu().double()
    t = 0.5 * (x64[:, :, None, :] * a64[:, None]).sum(-1)
    own = (t[..., None] * b64[:, None, :r]).sum(2) + 0.5 * b64[:, None, r]
    want = (x64[..., None] * w64).sum(2) + own
    for kind in (torch.isposinf, torch.isneginf, torch.isnan):
        assert bool(kind(want).any())
        wrong = int((kind(y) != kind(want)).sum())
        assert wrong == 0, kind.__name__


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("per", [1, 16])
def test_intermediates_at_the_top_of_the_range(device, dtype, per):
    """x A^T between bfloat16's and float32's largest value is finite, and so is its product with a small B."""
    pop, n_in, n_out = 32, 64, 128
    x = torch.zeros(pop, per, n_in, dtype=dtype, device=device)
    x[..., :2] = 2.0 ** 64
    a = torch.zeros(pop, 1, n_in, dtype=dtype, device=device)
    a[..., 0], a[..., 1] = 1.9921875 * 2.0 ** 63, 1.5625 * 2.0 ** 55      # together 1.9982910 2^127: rounds to infinity in 8 bits
    b = torch.full((pop, 1, n_out), 2.0 ** -120, dtype=dtype, device=device)
    weight = torch.zeros(n_in, n_out, dtype=dtype, device=device)
    want = 1.9921875 * 2.0 ** 7 + 1.5625 / 2
    y = lowrank_linear(x, weight, a, b).double()
    assert float((y - want).abs().max()) <= want * (torch.finfo(dtype).eps / 2 + 8 * U)


# ------------------------------------------------------------------ networks

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hidden,final", [("gelu", "tanh"), ("relu", "gelu"), (torch.sin, lambda v: 2 * v), (torch.nn.functional.silu, "sigmoid")])
def test_networks_of_any_activation(device, dtype, hidden, final):
    """MLP's other activations, by name and as callables: the layers' bound of test_linear, each layer on the one before as it came
    out, then an activation whose slope is below 2 here and which rounds twice (to its type, and once inside)."""
    gen = torch.Generator().manual_seed(37)
    net = MLP([12, 40, 5], activation=hidden, final_activation=final)
    center = net.init(rnd.PRNGKey(3)).to(device)
    factors = randn(gen, 9, net.lowrank_size(2), dtype=dtype).to(device)
    x = randn(gen, 9, 4, 12, dtype=dtype).to(device)
    y = net.lowrank_apply(center, factors, x, 2, 0.1)
    assert y.shape == (9, 4, 5) and y.dtype == dtype
    names = {"gelu": torch.nn.functional.gelu, **ACT}
    (a0, b0), (a1, b1) = net.lowrank_factors(factors, 2)
    w0, c0, w1, c1 = (v.to(t) for v, t in zip(center.split([480, 40, 200, 5]), (dtype, torch.float32) * 2))
    act, fin = (names.get(v, v) for v in (hidden, final))
    eps = torch.finfo(dtype).eps / 2
    h = lowrank_linear(x, w0.view(12, 40), a0, b0, bias=c0, scale=0.1, activation=hidden if hidden in ACT else "identity")
    h = h if hidden in ACT else act(h)
    z, off = linear_oracle(h, w1.view(40, 5), a1, b1, bias=c1, scale=0.1)
    want = fin(z)
    bound = 2 * off + (3 if final in ACT else 4) * eps * (want.abs() + 2 * off) + 16 * U
    assert bool(((y.cpu().double() - want).abs() <= bound).all())
    one = net.lowrank_apply(center, factors, x[:3, 0], 2, 0.1, index=torch.tensor([2, -1, 0], device=device))
    assert one.shape == (3, 5) and one.dtype == dtype


# ------------------------------------------------------------------ every variant that a size chooses

ANY, FEW, GROUPED = 0, 1, 1000                     # any-size tiles, up to four rows, individuals' parts in the tiles
BF, FP = torch.bfloat16, torch.float32
VARIANTS = [  # type, individuals, rows each (None: rows that name their individual), in, out, rank, kernel: rows of its tile (+ GROUPED)
    # bf16 tiles of 256: 2 to 5 steps of K and more, a last step in part, odd tile edges; 1 to 8 individuals in a tile
    (BF, 256, 256, 64, 256, 16, GROUPED + 256),     # one individual a tile
    (BF, 683, 48, 72, 264, 5, GROUPED + 256),       # three fragments each: up to seven individuals, which straddle tiles
    (BF, 2048, 32, 96, 248, 16, GROUPED + 256),     # eight individuals a tile
    (BF, 1500, 23, 128, 264, 3, GROUPED + 256),     # two fragments, the last one in part
    (BF, 300, 230, 160, 132, 7, GROUPED + 256),     # fifteen fragments
    (BF, 66, 1000, 200, 136, 16, GROUPED + 256),    # individuals longer than a tile
    (BF, 3, 22000, 264, 136, 1, GROUPED + 256),
    (BF, 683, 48, 73, 259, 5, GROUPED + 256),       # rows off 16 bytes: copied
    (BF, 33000, 1, 64, 264, 3, 256),
    (BF, 66000, 1, 104, 136, 1, 256),
    (BF, 130, 256, 136, 264, 17, 256),              # rank above 16
    (BF, 12, None, 264, 264, 4, 256),
    (BF, 12, None, 1096, 1032, 4, 256),
    (BF, 12, None, 265, 259, 4, 256),
    # tiles of 128
    (BF, 256, 128, 64, 128, 16, GROUPED + 128),
    (BF, 2100, 16, 72, 120, 9, GROUPED + 128),      # eight individuals a tile
    (BF, 2100, 16, 96, 264, 9, GROUPED + 128),      # sixteen would meet in a tile of 256
    (BF, 700, 48, 104, 66, 2, GROUPED + 128),
    (BF, 33000, 1, 200, 72, 3, 128),
    (BF, 900, 20, 72, 200, 20, 128),
    (FP, 256, 128, 32, 128, 16, GROUPED + 128),
    (FP, 2100, 16, 36, 120, 9, GROUPED + 128),
    (FP, 230, 48, 68, 264, 5, GROUPED + 128),
    (FP, 40, 300, 100, 260, 12, GROUPED + 128),
    (FP, 40, 300, 499, 261, 12, GROUPED + 128),
    (FP, 11000, 1, 132, 264, 2, 128),
    (FP, 5, None, 260, 264, 3, 128),
    (FP, 100, 330, 64, 72, 24, 128),
    # tiles of 64, K whole and divided, and of 16
    (BF, 40, 48, 136, 72, 16, GROUPED + 64), (FP, 40, 48, 68, 72, 16, GROUPED + 64), (BF, 500, 23, 72, 40, 3, GROUPED + 64),
    (BF, 20000, 1, 72, 64, 3, 64), (FP, 20000, 1, 72, 60, 3, 64),                        # t by the tiles' own workgroups
    (BF, 300, 1, 1096, 200, 5, 64), (FP, 300, 1, 1096, 200, 5, 64),
    (BF, 16, 1, 520, 264, 5, 16), (FP, 3, 5, 520, 264, 20, 16), (BF, 9, 1, 72, 1000, 5, 16),
    # up to four rows, any size
    (BF, 4, 1, 1001, 264, 5, FEW), (FP, 1, 1, 300, 1004, 5, FEW), (BF, 300, 7, 11, 32, 1, ANY), (FP, 300, 7, 11, 32, 1, ANY),
]


def kernel_of(dtype, pop, per, n_in, n_out, r):
    rows = 33003 if per is None else pop * per
    at, dims, ints = host_call((rows, pop, per or 1, (per or 1) * n_in, n_in, r * n_in, r * n_out),
                               (n_in, n_out, r, 0, 0, int(dtype == torch.bfloat16), 2 * (per is None)))
    return _native.hip().evox_hip_lowrank_linear_kernel(at, at, at, at, None, at, at, ctypes.addressof(dims), ctypes.addressof(ints))


@needs_library
@pytest.mark.parametrize("case", VARIANTS, ids=str)
def test_kernel_of_each_shape(case):
    """The shapes above take the kernels that they are there for."""
    *shape, kernel = case
    assert kernel_of(*shape) == kernel


@pytest.mark.gpu
@pytest.mark.parametrize("case", VARIANTS, ids=str)
def test_each_linear_kernel(cuda, case):
    dtype, pop, per, n_in, n_out, r, _ = case
    gen = torch.Generator().manual_seed(pop + n_in + n_out)
    for own_bias, act in ((0, "identity"), (1, "tanh")):
        weight, a, b = layer(gen, pop, n_in, n_out, r, own_bias, dtype, cuda, pitch=-(r * n_in + (r + own_bias) * n_out) % 8)
        kw = dict(bias=randn(gen, n_out).to(cuda) if own_bias else None, scale=0.4, activation=act)
        if per is None:
            kw["index"] = torch.randint(-1, pop, (33003,), generator=gen).to(cuda)
            x = randn(gen, 33003, n_in, dtype=dtype).to(cuda)
        else:
            x = randn(gen, pop, per, n_in, dtype=dtype).to(cuda)
        y = lowrank_linear(x, weight, a, b, **kw)
        check_linear(y, x, weight, a, b, **kw)
        assert torch.equal(y, lowrank_linear(x, weight, a, b, **kw))


SUM_VARIANTS = [  # type, individuals, in, out, rank, rows of the tile (0: any size)
    (BF, 64, 1024, 720, 1, 256), (BF, 40, 1000, 1000, 2, 256), (BF, 33, 1032, 700, 5, 256), (BF, 700, 768, 1024, 3, 256),
    (BF, 5000, 1024, 720, 1, 256), (BF, 4096, 1000, 700, 4, 256), (BF, 50, 1024, 768, 33, 256), (BF, 24, 1024, 720, 3, 256),
    (BF, 64, 64, 64, 1, 128), (BF, 33, 136, 264, 3, 128), (BF, 9000, 130, 136, 2, 128), (BF, 20000, 128, 128, 1, 128),
    (BF, 300, 300, 260, 16, 128), (BF, 300, 249, 250, 40, 128),
    (FP, 64, 64, 64, 1, 128), (FP, 33, 136, 264, 3, 128), (FP, 9000, 130, 136, 2, 128), (FP, 300, 1024, 720, 7, 128), (FP, 300, 251, 249, 40, 128),
    (BF, 300, 47, 400, 3, 0), (FP, 20000, 11, 32, 1, 0),
]


def sum_kernel_of(dtype, pop, n_in, n_out, r):
    at, dims, ints = host_call((pop, r * n_in, r * n_out), (n_in, n_out, r, int(dtype == torch.bfloat16)))
    return _native.hip().evox_hip_lowrank_sum_kernel(at, at, at, at, None, ctypes.addressof(dims), ctypes.addressof(ints))


@needs_library
@pytest.mark.parametrize("case", SUM_VARIANTS, ids=str)
def test_kernel_of_each_sum(case):
    *shape, kernel = case
    assert sum_kernel_of(*shape) == kernel


@pytest.mark.gpu
@pytest.mark.parametrize("case", SUM_VARIANTS, ids=str)
def test_each_sum_kernel(cuda, case):
    dtype, pop, n_in, n_out, r, _ = case
    gen = torch.Generator().manual_seed(pop + n_in + n_out)
    for own_bias in (0, 1):
        _, a, b = layer(gen, pop, n_in, n_out, r, own_bias, dtype, cuda, pitch=-(r * n_in + (r + own_bias) * n_out) % 8)
        w = randn(gen, pop).to(cuda)
        got = lowrank_weighted_sum(w, a, b, scale=-0.3)
        check_sum(got, w, a, b, -0.3)
        again = lowrank_weighted_sum(w, a, b, scale=-0.3)
        assert torch.equal(got[0], again[0]) and (not own_bias or torch.equal(got[1], again[1]))


@pytest.mark.gpu
def test_recorded_large_calls(cuda):
    """Large tiles recorded without a call before, replayed on new data with eager calls between the replays, on two graphs in turn."""
    gen = torch.Generator().manual_seed(41)
    sets = []
    for k in range(2):
        weight, a, b = layer(gen, 256, 128, 256, 16, 1, BF, cuda)
        _, sa, sb = layer(gen, 2000, 1024, 720, 4, 1, BF, cuda)
        sets.append((randn(gen, 256, 256, 128, dtype=BF).to(cuda), weight, a, b, randn(gen, 2000).to(cuda), sa, sb))

    def calls(x, weight, a, b, w, sa, sb):
        return (lowrank_linear(x, weight, a, b, activation="tanh"), *lowrank_weighted_sum(w, sa, sb))

    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(calls(*s))
    for _ in range(3):
        for s, graph, out in zip(sets, graphs, outs):
            s[0].copy_(randn(gen, 256, 256, 128, dtype=BF))
            s[4].copy_(randn(gen, 2000))
            want = calls(*s)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, want))
    # and both at once, each on a stream of its own
    want = [calls(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(calls(*s))
    torch.cuda.synchronize()
    for k, one in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(one, want[k % 2]))


@pytest.mark.gpu
def test_one_row_of_2_to_30_inputs(cuda):
    """Zeros but for a few inputs, the last among them."""
    n = 2 ** 30
    at = torch.tensor([0, 1, 127, 128, 2 ** 29 + 3, n - 1], device=cuda)
    gen = torch.Generator().manual_seed(43)
    few = [randn(gen, 1, 6, dtype=BF).to(cuda), randn(gen, 6, 8, dtype=BF).to(cuda), randn(gen, 1, 2, 6, dtype=BF).to(cuda)]
    x, weight, a = (torch.zeros(s, dtype=BF, device=cuda) for s in ((1, n), (n, 8), (1, 2, n)))
    x[:, at], weight[at], a[:, :, at] = few
    b = randn(gen, 1, 3, 8, dtype=BF).to(cuda)
    check_linear(lowrank_linear(x, weight, a, b), few[0], few[1], few[2], b)
