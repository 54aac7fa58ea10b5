"""The kernels of the local training step (group norm with activation, linear
with its epilogue, AdamW) against plain implementations in 64 bits.

Tolerances are the roundings themselves: u = 2^-24 for an operation in fp32,
``half`` a rounding to the output's type, times the magnitudes that enter an
operation. Sums over a group run over at most 64 dependent additions (rows of
a thread, lanes, waves, chunks); a product's sum over k is allowed k of them.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from murmura_amd import ops
from murmura_amd.ops import reference as ref

U = 2.0 ** -24
DEPTH = 64  # dependent roundings of a sum over a group, and of what leads to it
SLOPE = 1.13  # the largest derivative of the activations; none bends by more
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _require_native():
    assert ops.native_available(), "HIP extension must be present"


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _randn(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)


def _within(got, want, tol):
    err = (got.double().cpu() - want).abs()
    worst = (err - tol).max().item() if err.numel() else -1.0
    assert got.shape == want.shape
    assert worst <= 0, f"off by {worst:.3g} more than allowed (error {err.max().item():.3g})"


# ------------------------------------------------------------- group norm
def _gn_check(x, groups, w, b, act, res, dy, eps=1e-5, run=None):
    """x, w, b, res, dy on the CPU in their types; run makes the device's results."""
    dtype = x.dtype
    d = {k: None if t is None else t.double() for k, t in dict(x=x, w=w, b=b, res=res).items()}
    n, c = x.shape[:2]

    def rows(t):
        return t.reshape(n, groups, -1)

    def chan(t):
        return t.view((1, c) + (1,) * (x.dim() - 2)).expand(x.shape)

    one = torch.ones(c, dtype=torch.float64)
    ga, be = chan(one if w is None else d["w"]), chan(0 * one if b is None else d["b"])
    mu = rows(d["x"]).mean(2, keepdim=True)
    rs = 1 / (rows(d["x"] - mu.expand_as(rows(d["x"])).reshape(x.shape)).square().mean(2, keepdim=True) + eps).sqrt()
    mu, rs = (t.expand(n, groups, max(1, rows(d["x"]).shape[2])).reshape(x.shape) for t in (mu, rs))
    xhat = (d["x"] - mu) * rs
    a = (d["x"].abs() + mu.abs()) * rs + 1
    z = xhat * ga + be + (0 if res is None else d["res"])
    ez = DEPTH * U * (a * ga.abs() + be.abs() + (0 if res is None else d["res"].abs()))
    if act == "relu" and dy is not None:  # no derivative at the kink: nothing comes back there
        dy = dy.masked_fill(z.abs() <= 2 * ez, 0)
    leaves = [t.to("cuda").requires_grad_(dy is not None) for t in (x, w, b, res) if t is not None]
    it = iter(leaves)
    dev = [None if t is None else next(it) for t in (x, w, b, res)]
    y = ops.group_norm_act(dev[0], groups, dev[1], dev[2], eps, act, dev[3])
    zl = z.clone().requires_grad_(True)
    want = ref._activate(zl, act)
    assert y.dtype == dtype
    _within(y.detach(), want.detach(), SLOPE * ez + _half(dtype) * want.detach().abs() + 8 * U * want.detach().abs())
    if dy is None:
        return
    dd = dy.double()
    dz, = torch.autograd.grad(want, zl, dd)
    edz = dd.abs() * (SLOPE * ez + 8 * U * SLOPE)
    got = dict(zip([k for k, t in zip(("x", "w", "b", "res"), dev) if t is not None],
                   torch.autograd.grad(y, leaves, dy.to("cuda"))))

    def avg(t):
        return rows(t).mean(2, keepdim=True).expand_as(rows(t)).reshape(x.shape)

    gz = dz * ga
    dx = rs * (gz - avg(gz) - xhat * avg(gz * xhat))
    eg, ex = edz * ga.abs(), DEPTH * U * a
    tol = rs * (eg + avg(eg) + xhat.abs() * avg(eg * xhat.abs() + gz.abs() * ex) + ex * avg((gz * xhat).abs())
                + DEPTH * U * (gz.abs() + avg(gz.abs()) + xhat.abs() * avg((gz * xhat).abs())))
    _within(got["x"], dx, tol + _half(dtype) * dx.abs())
    sums = [0] + list(range(2, x.dim()))
    if w is not None:
        want = (dz * xhat).sum(sums)
        tol = (edz * xhat.abs() + dz.abs() * ex + DEPTH * U * (dz * xhat).abs()).sum(sums)
        _within(got["w"], want, tol + _half(w.dtype) * want.abs())
        assert got["w"].dtype == w.dtype
    if b is not None:
        want = dz.sum(sums)
        _within(got["b"], want, (edz + DEPTH * U * dz.abs()).sum(sums) + _half(b.dtype) * want.abs())
    if res is not None:
        _within(got["res"], dz, edz + _half(dtype) * dz.abs())


GN_SHAPES = [
    ((2, 64, 8, 8), 32), ((3, 60, 7, 5), 5), ((1, 6, 1, 1), 3), ((5, 7, 3, 3), 7), ((2, 1030, 4, 4), 1),
    ((2, 36, 33, 31), 9), ((4, 24), 3), ((3, 5), 5), ((1, 8, 70, 70), 2), ((2, 512, 9, 9), 16),
    ((1, 3, 64, 64), 1), ((2, 96, 40, 3), 2), ((2, 12, 1, 300), 12), ((1, 64, 150, 140), 8), ((9, 32, 70, 75), 2),
    ((130, 8, 130, 131), 2), ((3, 640, 6, 6), 8), ((1, 1600, 5, 5), 1),
]


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("act", ref.ACTIVATIONS)
@pytest.mark.parametrize("shape,groups", GN_SHAPES)
def test_group_norm_act(shape, groups, act, dtype):
    c, seed = shape[1], 31 * GN_SHAPES.index((shape, groups))
    x = (_randn(shape, FP32, seed) * 1.7 + _randn((1, c) + (1,) * (len(shape) - 2), FP32, seed + 1)).to(dtype)
    w, b = (1 + 0.3 * _randn((c,), FP32, seed + 2)).to(dtype), _randn((c,), dtype, seed + 3)
    res = _randn(shape, dtype, seed + 4) if act in ("relu", "gelu") else None
    _gn_check(x, groups, w, b, act, res, _randn(shape, dtype, seed + 5))


def test_group_norm_parameters_in_fp32_or_absent():
    x, dy = _randn((2, 16, 5, 5), BF16, 1), _randn((2, 16, 5, 5), BF16, 2)
    w, b = 1 + 0.1 * _randn((16,), FP32, 3), _randn((16,), FP32, 4)
    _gn_check(x, 4, w, b, "silu", None, dy)
    _gn_check(x, 4, None, None, "silu", dy, dy)
    _gn_check(x, 4, w, None, "none", None, dy)
    _gn_check(x, 4, None, b, "relu", None, dy)
    _gn_check(x, 4, w, b, "gelu", None, None)


def test_group_norm_level_far_above_spread():
    # a level of 1000 around a spread of 1, one outlier at the first pixel
    x = 1000 + _randn((2, 8, 20, 20), FP32, 5)
    x[:, :, 0, 0] = -5000
    _gn_check(x, 2, None, None, "none", None, _randn(x.shape, FP32, 6))


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_group_norm_layouts(dtype):
    w, b = _randn((24,), dtype, 1).cuda(), _randn((24,), dtype, 2).cuda()
    base = _randn((2, 6, 7, 24), dtype, 3).cuda()
    cl = base.permute(0, 3, 1, 2)
    want = ops.group_norm_act(cl, 4, w, b, act="silu")
    assert want.is_contiguous(memory_format=torch.channels_last)
    wide = torch.randn(2, 6, 9, 24, device="cuda").to(dtype).permute(0, 3, 1, 2)
    wide[:, :, :, 1:8] = cl
    off = torch.empty(base.numel() + 1, device="cuda", dtype=dtype)[1:].view_as(base).copy_(base)
    for x in (cl.contiguous(), wide[:, :, :, 1:8], torch.stack([cl, cl], 4)[..., 0]):
        assert torch.equal(ops.group_norm_act(x, 4, w, b, act="silu"), want)
    # off the 16 bytes rows are split among the threads otherwise, and sums run in another order:
    # both are within DEPTH * U of what enters (values here are at most 5, a deviation at least 0.8),
    # and a rounding apart
    near = ops.group_norm_act(off.permute(0, 3, 1, 2), 4, w, b, act="silu")
    enters = 2 * 5 / 0.8 * w.abs().max() + b.abs().max()
    assert ((near.float() - want.float()).abs()
            <= 2 * SLOPE * DEPTH * U * enters + 2 * _half(dtype) * want.float().abs()).all()
    # a gradient that is one value everywhere has strides of zero
    x = cl.detach().requires_grad_(True)
    g1, = torch.autograd.grad(ops.group_norm_act(x, 4, w, b, act="silu").float().sum(), x)
    g2, = torch.autograd.grad(ops.group_norm_act(x, 4, w, b, act="silu"), x, torch.ones_like(cl))
    assert torch.equal(g1, g2)


def test_group_norm_empty_and_nan():
    w = torch.ones(4, device="cuda", requires_grad=True)
    for shape in ((0, 4, 3, 3), (2, 4, 0, 3), (0, 4)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = ops.group_norm_act(x, 2, w)
        assert y.shape == x.shape
        dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
        assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))
    # what is not a number stays within its own group of its own sample
    x = _randn((2, 4, 6, 6), FP32, 1).cuda()
    x[1, 0, 2, 2] = math.nan
    for act in ref.ACTIVATIONS:
        bad = torch.isnan(ops.group_norm_act(x, 2, act=act))
        assert bad[1, :2].all() and not bad[0].any() and not bad[1, 2:].any()


def test_group_norm_repeats_and_places_past_31_bits():
    # 2.2e9 values: the last sample against the same sample alone
    n = 2 ** 31 // (8 * 64 * 64) + 3
    x = torch.empty((n, 64, 64, 8), device="cuda", dtype=BF16).normal_().permute(0, 3, 1, 2).requires_grad_(True)
    y = ops.group_norm_act(x, 2, act="silu")
    dx, = torch.autograd.grad(y, x, x.detach())
    last = x.detach()[-1:].clone(memory_format=torch.channels_last).requires_grad_(True)
    z = ops.group_norm_act(last, 2, act="silu")
    dz, = torch.autograd.grad(z, last, last.detach())
    assert torch.equal(y[-1:], z) and torch.equal(dx[-1:], dz)


# ----------------------------------------------------------------- linear
def _linear_check(x, w, b, act, res, dy):
    dtype, k = x.dtype, x.shape[-1]
    xd, wd = x.double().reshape(-1, k), w.double()
    n, m = w.shape[0], xd.shape[0]
    z = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    for t in (b, res):
        if t is not None:
            z = z + t.double().reshape(-1, n)
            mag = mag + t.double().abs().reshape(-1, n)
    ez = (k + 8) * U * mag
    if act == "relu" and dy is not None:
        dy = dy.masked_fill((z.abs() <= 2 * ez).view(dy.shape), 0)
    leaves = [t.to("cuda").requires_grad_(dy is not None) for t in (x, w, b, res) if t is not None]
    it = iter(leaves)
    dev = [None if t is None else next(it) for t in (x, w, b, res)]
    y = ops.linear_act(dev[0], dev[1], dev[2], act, dev[3])
    assert y.dtype == dtype and y.shape == (*x.shape[:-1], n)
    zl = z.clone().requires_grad_(True)
    want = ref._activate(zl, act)
    wv = want.detach()
    _within(y.detach().reshape(m, n), wv, SLOPE * ez + (8 * U + _half(dtype)) * wv.abs())
    if dy is None:
        return
    dd = dy.double().reshape(m, n)
    dz, = torch.autograd.grad(want, zl, dd)
    # silu and gelu see z in the operands' type; dz is rounded to it for the products
    ekeep = ez + (_half(dtype) * (z.abs() + ez) if act in ("silu", "gelu") else 0)
    edz = dd.abs() * (SLOPE * ekeep + 8 * U * SLOPE)
    eround = edz + (_half(dtype) * (dz.abs() + edz) if act != "none" else 0)
    got = dict(zip([k for k, t in zip(("x", "w", "b", "res"), dev) if t is not None],
                   torch.autograd.grad(y, leaves, dy.to("cuda"))))
    dx = dz @ wd
    tol = eround @ wd.abs() + (n + 8) * U * (dz.abs() @ wd.abs())
    _within(got["x"].reshape(m, k), dx, tol + _half(dtype) * (dx.abs() + tol))
    dw = dz.t() @ xd
    tol = eround.t() @ xd.abs() + (m + 8) * U * (dz.abs().t() @ xd.abs())
    _within(got["w"], dw, tol + _half(dtype) * (dw.abs() + tol))
    if b is not None:
        db = dz.sum(0)
        tol = (edz + (m + 8) * U * dz.abs()).sum(0)
        _within(got["b"], db, tol + _half(b.dtype) * (db.abs() + tol))
    if res is not None:
        _within(got["res"].reshape(m, n), dz, eround)


LINEAR_SHAPES = [
    (600, 1500, 1000), (34, 42, 66), (258, 262, 514), (2050, 2002, 1950), (1023, 1031, 1029), (1300, 700, 1100), (8, 8200, 520), (1500, 64, 1600),
    (1, 1, 1), (1, 64, 128), (1, 561, 250), (3, 33, 65), (7, 8, 16), (16, 512, 96), (17, 100, 10), (64, 3136, 64),
    (64, 128, 62), (65, 129, 127), (130, 64, 257), (300, 72, 200), (257, 512, 264), (2, 4000, 130), (520, 40, 512),
    (512, 192, 520),
]


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("act", ref.ACTIVATIONS)
@pytest.mark.parametrize("m,k,n", LINEAR_SHAPES)
def test_linear_act(m, k, n, act, dtype):
    seed = 17 * LINEAR_SHAPES.index((m, k, n))
    x, w = _randn((m, k), dtype, seed), (_randn((n, k), FP32, seed + 1) / math.sqrt(k)).to(dtype)
    b = _randn((n,), dtype, seed + 2)
    res = _randn((m, n), dtype, seed + 3) if act in ("none", "gelu") else None
    _linear_check(x, w, b, act, res, _randn((m, n), dtype, seed + 4))


def test_linear_leading_sizes_and_missing_parts():
    w = _randn((20, 12), BF16, 1)
    for lead in ((), (3,), (2, 3), (2, 1, 4)):
        x, dy = _randn((*lead, 12), BF16, 2), _randn((*lead, 20), BF16, 3)
        _linear_check(x, w, None, "gelu", None, dy)
        _linear_check(x, w, _randn((20,), FP32, 4), "silu", dy, dy)
        _linear_check(x, w, None, "relu", None, None)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_linear_layouts(dtype):
    x, w, b = _randn((70, 40), dtype, 1).cuda(), _randn((48, 40), dtype, 2).cuda(), _randn((48,), dtype, 3).cuda()
    want = ops.linear_act(x, w, b, "silu")
    wide = torch.full((70, 90), math.nan, device="cuda", dtype=dtype)
    wide[:, 3:43] = x
    off = torch.full((48 * 41 + 1,), math.nan, device="cuda", dtype=dtype)[1:].view(48, 41)
    off[:, :40] = w
    # rows off the 16 bytes may be summed by another kernel, in another order: both are within
    # (k + 8) U of the products' magnitudes, and a rounding apart
    mag = (x.float().abs() @ w.float().abs().t() + b.float().abs()).double()
    tol = SLOPE * 2 * (40 + 8) * U * mag + 2 * _half(dtype) * want.double().abs()
    for xx in (x, wide[:, 3:43], x.t().contiguous().t()):
        for ww in (w, off[:, :40], w.t().contiguous().t()):
            assert ((ops.linear_act(xx, ww, b, "silu").double() - want.double()).abs() <= tol).all()
    # one row for all: strides of zero
    row = ops.linear_act(x[:1].expand(5, 40), w, b, "silu")
    assert torch.equal(row, row[:1].expand(5, 48))
    xr = x.detach().requires_grad_(True)
    g1, = torch.autograd.grad(ops.linear_act(xr, w, b).float().sum(), xr)
    g2, = torch.autograd.grad(ops.linear_act(xr, w, b), xr, torch.ones_like(want))
    assert torch.equal(g1, g2)


def test_linear_empty_and_nan():
    for m, k, n in ((0, 4, 3), (5, 0, 3), (5, 4, 0)):
        x = torch.zeros(m, k, device="cuda", requires_grad=True)
        w = torch.zeros(n, k, device="cuda", requires_grad=True)
        b = torch.ones(n, device="cuda", requires_grad=True)
        y = ops.linear_act(x, w, b, "silu")
        assert torch.equal(y, torch.nn.functional.silu(b).detach().expand(m, n))
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert torch.equal(dx, torch.zeros_like(x)) and torch.equal(dw, torch.zeros_like(w))
        assert db.shape == b.shape and (m > 0 or torch.equal(db, torch.zeros_like(b)))
    x, w = _randn((9, 40), BF16, 1).cuda(), _randn((33, 40), BF16, 2).cuda()
    x[4, 39] = math.inf
    w[7, 39] = 0
    for act in ref.ACTIVATIONS:
        bad = ~torch.isfinite(ops.linear_act(x, w, act="none"))
        assert bad[4].all() and not bad[:4].any() and not bad[5:].any()


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_linear_against_differences(dtype):
    # phi(t) = <y(x + t a, w + t c), dy> has the derivative <dx, a> + <dw, c>: in fp32 a step of
    # 2^-6 leaves (third derivative)/6 * 2^-12 and 2^-24/2^-6 of the sums' magnitude
    if dtype == BF16:
        pytest.skip("a step that bf16 resolves is no small one")
    x, w, dy = _randn((33, 40), dtype, 1).cuda(), (0.1 * _randn((50, 40), dtype, 2)).cuda(), _randn((33, 50), dtype, 3).cuda()
    a, c = _randn((33, 40), dtype, 4).cuda(), (0.1 * _randn((50, 40), dtype, 5)).cuda()
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(ops.linear_act(xr, wr, act="gelu"), (xr, wr), dy)
    slope = (dx.double() * a).sum() + (dw.double() * c).sum()
    t = 2.0 ** -6
    phi = [(ops.linear_act(x + s * a, w + s * c, act="gelu").double() * dy).sum() for s in (t, -t)]
    mag = (ops.linear_act(x.abs(), w.abs(), act="none").double() * dy.abs()).sum()
    # gelu's third derivative stays below 2; dz/dt and d2z/dt2 by their magnitudes
    d1 = (ops.linear_act(a.abs(), w.abs()) + ops.linear_act(x.abs(), c.abs())).double()
    d2 = 2 * ops.linear_act(a.abs(), c.abs()).double()
    third = ((2 * d1 ** 3 + 3 * d1 * d2) * dy.abs()).sum()
    assert abs((phi[0] - phi[1]) / (2 * t) - slope) <= third * t * t / 6 + 48 * U * mag / t


# ------------------------------------------------------------------ AdamW
def _adamw_case(shapes, dtype, bits, seed, device, gtype=None):
    sizes = [math.prod(s) for s in shapes]
    total = sum(sizes)
    flat = (0.05 * _randn((total,), FP32, seed)).to(dtype).to(device)
    params = [p.view(s) for p, s in zip(flat.split(sizes), shapes)]
    grads = [(10.0 ** (i % 5 - 4) * _randn(s, FP32, seed + 1 + i)).to(gtype or dtype).to(device)
             for i, s in enumerate(shapes)]
    return flat, params, grads, ops.adamw_state(total, device, bits)


def _flat_state(m):
    return [m] if isinstance(m, torch.Tensor) else list(m)


ADAMW_SHAPES = [
    [(1,)], [(7,)], [(256,)], [(1000, 3)], [(3, 3), (257,), (1,), (0,), (64, 33), (5,)],
    [(2, 2)] * 400, [(1,)] * 3 + [(513,)] * 170 + [(4096,)], [(70001,), (63,), (8192,)],
]


@pytest.mark.parametrize("dtype,gtype", [(FP32, FP32), (BF16, BF16), (BF16, FP32)])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("shapes", ADAMW_SHAPES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_adamw_step(shapes, bits, dtype, gtype):
    """Moments: every operation is one rounding in both, so the bits are the
    same. Parameters: root and reciprocal are off by a unit (2 U) each, which
    with the roundings of three products stays below 8 U of the step (|m| <= 3.2
    sqrt(v) after so few steps, so a step is at most 5 lr); two sums round to U
    of a parameter below 1. In bf16 a value so near a border may go to the other
    side: 2^-8 of itself."""
    if bits == 8 and len(shapes) == 400:
        pytest.skip("refused: see test_adamw_refusals")
    cpu = _adamw_case(shapes, dtype, bits, 3, "cpu", gtype)
    gpu = _adamw_case(shapes, dtype, bits, 3, "cuda", gtype)
    for k in range(3):
        for _, params, grads, state in (cpu, gpu):
            ops.adamw_step(params, [g * (k + 1) for g in grads], *state, 1e-2, weight_decay=0.1, seed=k * 977 - 5)
    tol = 3 * (8 * U * 5 * 1e-2 + 2 * U)
    diff = (cpu[0].double() - gpu[0].cpu().double()).abs()
    if dtype == FP32:
        assert diff.max() <= tol
    else:
        assert (diff <= tol + 3 * 2.0 ** -8 * cpu[0].double().abs()).all()
        # the share of values within 24 U * 0.05 of a border that lie 2^-9 * 2^-5 apart at the least
        assert (diff > 0).sum() <= 3 + 0.01 * diff.numel()
    for a, b in zip(cpu[3][:2], gpu[3][:2]):
        for x, y in zip(_flat_state(a), _flat_state(b)):
            assert torch.equal(x, y.cpu())
    assert int(gpu[3][2]) == 3
    if bits == 8:
        for t in (FP32, BF16):
            for a, b in zip(ops.adamw_dequantize(*cpu[3][:2], dtype=t), ops.adamw_dequantize(*gpu[3][:2], dtype=t)):
                assert torch.equal(a, b.cpu())


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_flat_layouts_and_device_lr(bits):
    shapes = [(8, 3, 3, 3), (10,), (16, 8)]
    flat, params, grads, state = _adamw_case(shapes, BF16, bits, 5, "cuda")
    want = flat.clone()
    other = ops.adamw_state(flat.numel(), "cuda", bits)
    ops.adamw_step(params, grads, *state, 1e-2, seed=9)
    ops.adamw_step(want, torch.cat([g.reshape(-1) for g in grads]), *other,
                   torch.tensor([1e-2], device="cuda"), seed=9)
    # the number 1e-2 in 64 bits and in 32 differ by 2e-8 of itself: one value in some thousands may
    # round to the other side
    assert (flat != want).float().mean() < 0.02
    assert torch.equal(_flat_state(state[0])[0], _flat_state(other[0])[0])
    # channels-last parameters, their gradients with other strides, and off the 16 bytes
    buf = torch.zeros(8 * 27 + 1, device="cuda")
    p = buf[1:].view(8, 3, 3, 3).permute(0, 3, 1, 2)
    g = torch.randn(8, 3, 3, 3, device="cuda")
    one, two = ops.adamw_state(216, "cuda", bits), ops.adamw_state(216, "cuda", bits)
    q = torch.zeros(216, device="cuda")
    ops.adamw_step([p], [g], *one, 0.1)
    ops.adamw_step(q, g.permute(0, 2, 3, 1).reshape(-1), *two, 0.1)
    assert torch.equal(buf[1:], q) and buf[0] == 0
    assert torch.equal(_flat_state(one[0])[0], _flat_state(two[0])[0])


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_nan_and_inf_stay_where_they_are(bits):
    flat, params, grads, state = _adamw_case([(600,)], FP32, bits, 5, "cuda")
    clean = _adamw_case([(600,)], FP32, bits, 5, "cuda")
    grads[0][3], grads[0][300] = math.nan, math.inf
    for _ in range(2):
        ops.adamw_step(params, grads, *state, 1e-2)
        ops.adamw_step(clean[1], clean[2], *clean[3], 1e-2)
    bad = torch.zeros(600, dtype=torch.bool, device="cuda")
    bad[3] = bad[300] = True
    assert torch.isnan(flat[bad]).all()
    assert torch.isfinite(flat[~bad]).all()
    if bits == 32:
        assert torch.equal(flat[~bad], clean[0][~bad])


def test_adamw_places_past_31_bits():
    n = 2 ** 31 + 5001
    p = torch.zeros(n, device="cuda")
    g = torch.empty(n, device="cuda").uniform_(-1, 1)
    state = ops.adamw_state(n, "cuda", 8)
    ops.adamw_step([p[:1000], p[1000:]], [g[:1000], g[1000:]], *state, 1.0, weight_decay=0.0)
    # the first step moves every parameter by lr * g / (|g| + eps * ...): +-1 where |g| >> 1e-8
    tail = slice(n - 5001, None)
    sure = g[tail].abs() > 1e-3
    assert torch.allclose(p[tail][sure], -g[tail][sure].sign(), rtol=0, atol=2e-5)
    m, v = ops.adamw_dequantize((state[0][0][-5001:], state[0][1][-20:]), (state[1][0][-5001:], state[1][1][-20:]))
    # 3 bits of mantissa: an eighth of itself at most
    assert ((m - 0.1 * g[tail]).abs() <= 0.125 * 0.1 * g[tail].abs() + 2.0 ** -17).all()


def test_adamw_v_moves_by_less_than_its_steps():
    """With one gradient forever, v goes to g*g over thousands of steps of a
    thousandth each, though a code's steps are an eighth."""
    n = 4096
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.5, device="cuda")
    state = ops.adamw_state(n, "cuda", 8)
    for _ in range(3000):
        ops.adamw_step(p, g, *state, 1e-3, weight_decay=0.0)
    _, v = ops.adamw_dequantize(*state[:2])
    want = 0.25 * (1 - 0.999 ** 3000)
    # one value strays by sqrt(step * v / 2) = sqrt(0.125 / 2) v; of the mean of n, 5 of these / sqrt(n)
    assert abs(v.mean().item() / want - 1) < 5 * math.sqrt(0.125 / 2) / math.sqrt(n) + 1e-3


# ---------------------------------------------------------- all of a step
def _step_state(device):
    g = torch.Generator().manual_seed(3)

    def make(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g)).to(BF16).to(device)

    flat = torch.cat([make(16 * 8, scale=0.1), 1 + make(8, scale=0.1), make(8), make(40 * 72, scale=0.1), make(40)])
    x, target = make(12, 3, 3, 16), make(12, 40)
    return flat, x, target, ops.adamw_state(flat.numel(), device, 8)


def _one_step(flat, x, target, state):
    """A pixel-wise linear, group norm with relu, a linear with residual; AdamW over all."""
    sizes = [(8, 16), (8,), (8,), (40, 72), (40,)]
    params = [p.view(s).detach().requires_grad_(True)
              for p, s in zip(flat.split([math.prod(s) for s in sizes]), sizes)]
    h = ops.linear_act(x, params[0]).permute(0, 3, 1, 2)
    h = ops.group_norm_act(h, 2, params[1], params[2], act="relu").permute(0, 2, 3, 1)
    y = ops.linear_act(h.reshape(12, 72), params[3], params[4], act="silu", res=target)
    loss = (y.float() - 1).square().mean()
    grads = torch.autograd.grad(loss, params)
    ops.adamw_step([p.detach() for p in params], grads, *state, 1e-2, seed=4)
    return loss.detach()


def test_step_learns_and_repeats():
    a, b = _step_state("cuda"), _step_state("cuda")
    for k in range(5):
        la, lb = _one_step(*a), _one_step(*b)
        assert torch.equal(la, lb) and torch.equal(a[0], b[0])


def test_step_in_a_graph_beside_eager_steps():
    eager, other = _step_state("cuda"), _step_state("cuda")
    captured = _step_state("cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _one_step(*captured)
    torch.cuda.current_stream().wait_stream(side)
    _one_step(*eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = _one_step(*captured)
    for k in range(4):
        graph.replay()
        want = _one_step(*eager)
        _one_step(*other)  # eager work between replays, from the same allocator
        torch.cuda.synchronize()
        assert torch.equal(loss, want)
        assert torch.equal(captured[0], eager[0])
        assert int(captured[3][2]) == int(eager[3][2]) == k + 2


def test_step_on_another_stream():
    a, b = _step_state("cuda"), _step_state("cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            la = _one_step(*a)
    for _ in range(3):
        lb = _one_step(*b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(la, lb) and torch.equal(a[0], b[0])


def test_refusals_on_the_device():
    x = torch.randn(2, 8, 3, 3, device="cuda", requires_grad=True)
    y = ops.group_norm_act(x, 2)
    g, = torch.autograd.grad(y.sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.square().sum(), x, create_graph=True)
    w = torch.randn(4, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.linear_act(torch.randn(3, 8, device="cuda"), w).square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="fp32 or bf16"):
        ops.group_norm_act(x.double(), 2)
    with pytest.raises(RuntimeError, match="fp32 or bf16"):
        ops.linear_act(torch.randn(3, 8, device="cuda").half(), w.half())
    with pytest.raises(ValueError):
        ops.group_norm_act(x, 2, torch.ones(8))
    with pytest.raises(ValueError):
        ops.linear_act(torch.randn(3, 8), w)
    # an output changed in place is no longer what its gradient was made for
    y = ops.linear_act(torch.randn(3, 8, device="cuda"), w, act="relu")
    y.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), w)


def test_adamw_refusals():
    p, g = torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda")
    m, v, t = ops.adamw_state(10, "cuda")
    m8, v8, _ = ops.adamw_state(10, "cuda", 8)
    for args in (([p, p], [g, g], *ops.adamw_state(20, "cuda")), ([p], [g[:9]], m, v, t), ([p], [], m, v, t),
                 ([p], [g], m[:9], v, t), ([p], [g], m8, v, t), ([p], [g.cpu()], m, v, t), ([p], [g], m, v, t.int()),
                 ([p], [g.bfloat16()], m, v, t), ([p], [g], m.double(), v.double(), t), ([p[::2]], [g[::2]], m[:5], v[:5], t),
                 ([p[:1].expand(10)], [g], m, v, t), ([p[:6], p[4:]], [g[:6], g[4:]], *ops.adamw_state(12, "cuda"))):
        with pytest.raises(RuntimeError):
            ops.adamw_step(*args, 1e-3)
    with pytest.raises(RuntimeError, match="pass them as one"):
        many = torch.zeros(400, device="cuda")
        ops.adamw_step(list(many.split(1)), list(torch.zeros(400, device="cuda").split(1)), *ops.adamw_state(400, "cuda", 8), 1e-3)
    assert int(t) == 0 and not p.any()


# ----------------------------------------------------- a node's whole round
def _gpu_node(model, optimizer, dtype=BF16, shape=(3, 16, 16), n=48):
    from torch.utils.data import DataLoader, TensorDataset

    from murmura_amd.aggregation.fedavg import FedAvgAggregator
    from murmura_amd.core.node import Node

    data = TensorDataset(_randn((n, *shape), FP32, 9), torch.arange(n) % 4)
    loader = DataLoader(data, batch_size=16)
    return Node(0, model, loader, loader, FedAvgAggregator(), torch.device("cuda"), dtype=dtype,
                optimizer=optimizer)


@pytest.mark.parametrize("bits", [8, 32])
def test_node_rounds_with_group_norm_and_adamw(bits):
    from murmura_amd.core.optim import AdamWConfig
    from murmura_amd.models import ResNet18

    def train():
        torch.manual_seed(0)
        node = _gpu_node(ResNet18(num_classes=4, norm="group"), AdamWConfig(state_bits=bits))
        for r in range(3):  # captured once, replayed, between them a state from outside
            out = node.local_train(lr=1e-3, round_num=r)
            assert math.isfinite(out["loss"])
            node.set_state(node.get_state() * 0.99)
        assert int(node.optimizer.count) == 9  # warm-up steps are taken back
        return node

    a = train()
    assert torch.isfinite(a.get_state()).all()
    m = a.optimizer.tensors()[0]
    assert m.count_nonzero() > 0.5 * m.numel()


def test_graph_and_eager_node_take_the_same_steps(monkeypatch):
    """Fused MLP, AdamW in 32 bits: the captured epoch does what single steps do."""
    from murmura_amd.core.optim import AdamWConfig
    from murmura_amd.models import SimpleMLP

    def train(graphs):
        if not graphs:
            monkeypatch.setenv("MURMURA_NO_GRAPHS", "1")
        torch.manual_seed(0)
        node = _gpu_node(SimpleMLP(24, 64, 4, fused=True), AdamWConfig(), dtype=FP32, shape=(24,), n=16)
        for _ in range(4):
            node.local_train(lr=1e-2)  # one batch an epoch: its order does not matter to a sum
        monkeypatch.delenv("MURMURA_NO_GRAPHS", raising=False)
        return node

    a, b = train(True), train(False)
    assert int(a.optimizer.count) == int(b.optimizer.count) == 4
    # The captured epoch sums its 16 samples in another order: gradients differ by 16 * 24 U of
    # their magnitude. Adam divides by that magnitude, so 4 steps of 1e-2 differ by that share of
    # themselves, and by twice a whole step where a gradient is all rounding.
    diff = (a.get_state() - b.get_state()).abs()
    assert diff.max() <= 4 * 2 * 1e-2
    assert (diff > 4 * 1e-2 * 16 * 24 * U * 64).float().mean() < 0.02
