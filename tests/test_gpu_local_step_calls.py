"""Calls of the local training step's operators beside the ordinary ones."""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu

from murmura_amd import ops

U = 2.0 ** -24
BF16, FP32 = torch.bfloat16, torch.float32


def _randn(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)


def _within(got, want, tol):
    err = (got.double().cpu() - want).abs()
    worst = (err - tol).max().item()
    assert got.shape == want.shape
    assert worst <= 0, f"off by {worst:.3g} more than allowed (error {err.max().item():.3g})"


@pytest.mark.parametrize("lead", [(), (6,), (2, 3), (2, 1, 4)])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_inputs_changed_in_place_are_noticed(lead, act):
    base, w = _randn((*lead, 8), FP32, 1).cuda(), _randn((5, 8), FP32, 2).cuda().requires_grad_(True)
    # what the weight's gradient reads
    x = base.clone()
    y = ops.linear_act(x, w, act=act)
    x.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), w)
    # what the input's gradient reads
    x, v = base.clone().requires_grad_(True), w.detach().clone()
    y = ops.linear_act(x, v, act=act)
    v.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), x)
    # a copy that the call made of columns is its own
    x = base.new_zeros(*lead, 16)[..., ::2]
    x.copy_(base)
    want, = torch.autograd.grad(ops.linear_act(base, w, act=act).sum(), w)
    y = ops.linear_act(x, w, act=act)
    got, = torch.autograd.grad(y.sum(), w)
    assert torch.equal(got, want)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_refuses_before_it_changes_anything(bits):
    """The refusal of a later launch, and of what is looked at last."""
    def state(shapes):
        p = [_randn(s, FP32, i).cuda() for i, s in enumerate(shapes)]
        m, v, t = ops.adamw_state(sum(x.numel() for x in p), "cuda", bits)
        return p, [torch.ones_like(x) for x in p], m, v, t

    def refused(match, p, g, m, v, t, lr=1e-2):
        moments = [x for moment in (m, v) for x in ([moment] if isinstance(moment, torch.Tensor) else moment)]
        flat = [*p, *moments, t]
        kept, versions = [x.clone() for x in flat], [x._version for x in p]
        with pytest.raises(RuntimeError, match=match):
            ops.adamw_step(p, g, m, v, t, lr)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, flat))
        assert versions == [x._version for x in p]

    if bits == 8:  # 160 tensors fill the first launch, the next has over 160 within one scale
        refused("pass them as one", *state([(4096,)] * 160 + [(1,)] * 200))
    p, g, m, v, t = state([(300,), (20,)])
    refused("int64", p, g, m, v, t.int())
    refused("one fp32 value", p, g, m, v, t, torch.ones(2, device="cuda"))
    refused("parameter", p, g, m, ops.adamw_state(321, "cuda", bits)[1], t)
    refused("same bits", p, g, m, ops.adamw_state(320, "cuda", 40 - bits)[1], t)


def test_derivatives_going_forward_are_refused():
    def duals(call, *args):
        for i in range(len(args)):
            with fwd.dual_level():
                mixed = [fwd.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)]
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward"):
                        call(*mixed)

    x, w, b, r = (_randn(s, FP32, 1).cuda() for s in ((4, 8), (5, 8), (5,), (4, 5)))
    duals(lambda x, w, b, r: ops.linear_act(x, w, b, res=r), x, w, b, r)
    x, w, b, r = (_randn(s, FP32, 1).cuda() for s in ((2, 8, 3, 3), (8,), (8,), (2, 8, 3, 3)))
    duals(lambda x, w, b, r: ops.group_norm_act(x, 2, w, b, res=r), x, w, b, r)


def test_tracing_is_refused():
    """A trace would hold the result's memory and not the kernel that fills it."""
    from murmura_amd.ops.fused_linear import MurmuraLinear
    from murmura_amd.ops.fused_norm import MurmuraGroupNorm

    for module, x in ((MurmuraLinear(8, 5, act="relu"), _randn((3, 8), FP32, 1)),
                      (MurmuraGroupNorm(2, 8), _randn((3, 8), FP32, 1))):
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(module.cuda(), x.cuda(), check_trace=False)


def _scoring(model, shape, device, dtype=FP32, channels_last=True, classes=4):
    from torch.utils.data import DataLoader, TensorDataset

    from murmura_amd.aggregation.base import EvalContext
    from murmura_amd.core.flat import FlatParamStore

    store = FlatParamStore(model, torch.device(device), dtype, channels_last=channels_last)
    data = TensorDataset(_randn((24, *shape), FP32, 9), torch.arange(24) % classes)
    context = EvalContext(store, DataLoader(data, batch_size=24), torch.device(device))
    base = store.snapshot()
    return context, torch.stack([base, 0.9 * base, base + 0.01 * base.roll(1)])


@pytest.mark.parametrize("name", ["mlp", "wide", "femnist"])
def test_candidates_are_scored_in_one_graph(name):
    """All candidates through one captured, mapped forward, as without the fused layers, and as one
    by one: the fused layers run the same kernels, convolutions sum in another order (2^-24 times
    some thousand products, of a loss below 10)."""
    from murmura_amd.models import FEMNISTModel, SimpleMLP
    from murmura_amd.models.zoo import WideMLP

    torch.manual_seed(0)
    model, shape, tol = {
        "mlp": (lambda: SimpleMLP(12, fused=True), (12,), 64 * U),
        "wide": (lambda: WideMLP(12, 40, 4, fused=True), (12,), 64 * U),
        "femnist": (lambda: FEMNISTModel(hidden=64, num_classes=4, fused=True), (1, 28, 28), 4000 * U),
    }[name]
    context, states = _scoring(model(), shape, "cuda")
    batch = context.next_batch()
    for _ in range(3):
        got = context.losses_on_batch(states, batch)
        assert context._vmap_ok is True
        want = torch.stack([context.loss_on_batch(s, batch) for s in states])
        assert (got - want).abs().max() <= 10 * tol
        states = states.flip(0)


def test_candidates_with_group_norm_are_scored_one_by_one():
    """Which is faster (what each measured stands at EvalContext), and the same losses."""
    from murmura_amd.models import ResNet18

    torch.manual_seed(0)
    context, states = _scoring(ResNet18(num_classes=4, norm="group"), (3, 16, 16), "cuda")
    batch = context.next_batch()
    got = context.losses_on_batch(states, batch)
    assert context._vmap_ok is False and not context._graphs
    x, y = batch[0].contiguous(memory_format=torch.channels_last), batch[1]
    with torch.no_grad():
        mapped = context._ce_from_logits(context._stacked_call(states, x), y)
    # 20 layers of sums of up to 4608 products, of a loss below 10
    assert (got - mapped).abs().max() <= 10 * 20 * 4608 * U


def test_operators_under_vmap(device="cuda"):
    """Over the weights, over the input, over both, nested, and with gradients."""
    x, w, b = (_randn(s, FP32, i).to(device) for i, s in enumerate(((3, 4, 8), (3, 5, 8), (3, 5))))

    def f(x, w, b):
        return ops.linear_act(x, w, b, "silu")

    want = torch.stack([f(*t) for t in zip(x, w, b)])
    assert torch.equal(torch.vmap(f)(x, w, b), want)
    assert torch.equal(torch.vmap(f, (None, 0, 0))(x[0], w, b)[0], want[0])
    assert torch.equal(torch.vmap(f, (0, None, None))(x, w[0], b[0])[0], want[0])
    assert torch.equal(torch.vmap(f, (1, 1, 1), 1)(x.transpose(0, 1), w.transpose(0, 1), b.t()), want.transpose(0, 1))
    pairs = torch.vmap(torch.vmap(f, (None, 0, 0)), (0, None, None))(x, w, b)
    assert torch.equal(torch.stack([pairs[i, i] for i in range(3)]), want)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(torch.vmap(f)(*leaves).sum(), leaves)
    again = torch.autograd.grad(torch.stack([f(*t) for t in zip(*leaves)]).sum(), leaves)
    assert all(torch.equal(p, q) for p, q in zip(got, again))

    x, w, r = (_randn(s, FP32, i).to(device) for i, s in enumerate(((3, 2, 8, 3, 5), (3, 8), (2, 8, 3, 5))))

    def n(x, w):
        return ops.group_norm_act(x, 2, w, act="relu", res=r)

    want = torch.stack([n(*t) for t in zip(x, w)])
    assert torch.equal(torch.vmap(n)(x, w), want)
    assert torch.equal(torch.vmap(n, (None, 0))(x[0], w)[0], want[0])


def test_linear_over_more_rows_than_a_launch_has_blocks():
    """2^24 + 3 odd rows of bf16. All values are -1, 0 or 1, so that every sum is a whole number
    that fp32 holds: results are exact but for their own rounding."""
    m, k, n = 2 ** 24 + 3, 9, 8
    g = torch.Generator("cuda").manual_seed(1)
    x, w, dy = (torch.randint(-1, 2, s, generator=g, device="cuda").to(BF16) for s in ((m, k), (n, k), (m, n)))
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    y = ops.linear_act(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for rows in (slice(0, 1000), slice(m // 2, m // 2 + 1000), slice(m - 1000, m)):
        assert torch.equal(y[rows].float(), (x[rows].float() @ w.float().t()).to(BF16).float())
        assert torch.equal(dx[rows].float(), (dy[rows].float() @ w.float()).to(BF16).float())
    want = torch.stack([(dy * x[:, i:i + 1]).to(torch.int32).sum(0) for i in range(k)], 1)
    assert want.abs().max() < 2 ** 24 and torch.equal(dw, want.float().to(BF16))


def test_activations_in_fp32_hold_its_bits():
    """z * 1 is z, so y and dx are the activation and its derivative alone.

    erfc is within 4 units (8 u), its argument |z| sqrt(1/2) within 2 u, by which erfc changes at
    most z^2 + 1 times as much; exp within 1 unit, its argument z^2/2 within u; the reciprocal
    within 1 unit; a few products and sums of u each."""
    z = torch.cat([torch.linspace(-9, 9, 20011), torch.linspace(-80, 80, 20011)])
    x, one = z.view(-1, 1).cuda().requires_grad_(True), torch.ones(1, 1, device="cuda")
    for act in ("silu", "gelu"):
        y = ops.linear_act(x, one, act=act)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        d = z.double()
        if act == "silu":
            s, c = torch.sigmoid(d), torch.sigmoid(-d)
            t = 1 + d * c
            _within(y.detach().view(-1), d * s, 8 * U * (d * s).abs())
            _within(dx.view(-1), s * t, U * s * (8 * d.abs() + 2 + 8 * t.abs()))
            continue
        near = d.abs() <= 9  # beyond, erfc leaves the normal numbers
        cdf, pdf = 0.5 * torch.erfc(-d * math.sqrt(0.5)), torch.exp(-0.5 * d * d) / math.sqrt(2 * math.pi)
        _within(y.detach().view(-1)[near], (d * cdf)[near], U * ((2 * d * d + 12) * (d * cdf).abs())[near])
        _within(dx.view(-1)[near], (cdf + d * pdf)[near],
                U * ((2 * d * d + 12) * cdf + d.abs() * pdf * (d * d + 8))[near])
        assert torch.equal(y.detach().view(-1)[z.cuda() > 9], z.cuda()[z.cuda() > 9])
        assert y.detach().view(-1)[z.cuda() < -9].abs().max() < 1e-17


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,n", [
    (96, 64, 128), (65, 33, 71), (1, 8, 24), (300, 130, 66), (512, 512, 512), (1000, 1001, 999),
    (1030, 1024, 1018), (700, 4096, 1024), (4096, 256, 40),
])
def test_linear_keeps_the_activations_gradient(m, k, n, act):
    """Each row of x picks a row of W^T, so z is a value of W and exact in bf16, and of dx and dW
    there is left: dz in fp32 (the activation's derivative within 2^-20), its rest behind two halves
    of 8 bits, 2^-16, the products' sums, and one rounding to bf16."""
    half = torch.finfo(BF16).eps / 2
    pick = torch.randint(0, k, (m,), generator=torch.Generator().manual_seed(m + n))
    x = torch.nn.functional.one_hot(pick, k).to(BF16)
    w, dy = _randn((n, k), BF16, 1), _randn((m, n), BF16, 2)
    b = torch.zeros(n)
    z = (x.double() @ w.double().t()).requires_grad_(True)
    dz, = torch.autograd.grad(getattr(torch.nn.functional, act)(z), z, dy.double())
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(ops.linear_act(*leaves, act=act), leaves, dy.cuda())
    edz = 2.0 ** -20 * dy.double().abs()
    kept = edz + 2.0 ** -16 * (dz.abs() + edz)
    want, mag = dz @ w.double(), dz.abs() @ w.double().abs()
    tol = kept @ w.double().abs() + (2 * n + 8) * U * mag
    _within(dx, want, tol + half * (want.abs() + tol))
    want, mag = dz.t() @ x.double(), dz.abs().t() @ x.double()
    tol = kept.t() @ x.double() + (2 * m + 8) * U * mag
    _within(dw, want, tol + half * (want.abs() + tol))
    _within(db, dz.sum(0), (edz + (m + 8) * U * dz.abs()).sum(0))


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_linear_gradients_that_are_not_finite_stay_in_their_row(act):
    x, w, dy = _randn((70, 40), BF16, 1).cuda(), _randn((48, 40), BF16, 2).cuda(), _randn((70, 48), BF16, 3).cuda()
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    y = ops.linear_act(x, w, act=act)
    want, = torch.autograd.grad(y, x, dy, retain_graph=True)
    # the last of bf16's values: its dz is infinite, or is rounded to infinity, or neither
    dy[4, 7], dy[9, 3], dy[11] = math.inf, math.nan, torch.finfo(BF16).max
    dx, = torch.autograd.grad(y, x, dy)
    odd = torch.zeros(70, dtype=torch.bool, device="cuda")
    odd[[4, 9, 11]] = True
    assert torch.equal(dx[~odd], want[~odd])
    assert not torch.isfinite(dx[4]).any() and torch.isnan(dx[9]).all()


def _plain_loss(params, x, target):
    """A pixel-wise linear, group norm with relu, a linear with residual and silu."""
    f = torch.nn.functional
    h = f.linear(x, params[0]).permute(0, 3, 1, 2)
    h = torch.relu(f.group_norm(h.contiguous(), 2, params[1], params[2])).permute(0, 2, 3, 1)
    y = f.silu(f.linear(h.reshape(12, 72), params[3], params[4]) + target)
    return (y - 1).square().mean()


def test_a_step_goes_against_its_gradient():
    """The three operators together against the same step in 64 bits. AdamW's first step moves each
    parameter by lr against its gradient's sign; that is certain where a gradient is over a quarter of
    its tensor's largest: 64 roundings of bf16, 2^-8 each, all one way, would be needed to turn it."""
    sizes = [(8, 16), (8,), (8,), (40, 72), (40,)]
    flat = torch.cat([_randn((math.prod(s),), FP32, i) * (0.1 if i != 2 else 1) + (i == 1)
                      for i, s in enumerate(sizes)]).to(BF16)
    x, target = _randn((12, 3, 3, 16), BF16, 7), _randn((12, 40), BF16, 8)
    wide = [p.view(s).double().requires_grad_(True) for p, s in zip(flat.split([math.prod(s) for s in sizes]), sizes)]
    loss = _plain_loss(wide, x.double(), target.double())
    grads = torch.autograd.grad(loss, wide)

    dev = flat.cuda()
    state = ops.adamw_state(dev.numel(), "cuda", 8)
    params = [p.view(s).detach().requires_grad_(True) for p, s in zip(dev.split([math.prod(s) for s in sizes]), sizes)]
    h = ops.linear_act(x.cuda(), params[0]).permute(0, 3, 1, 2)
    h = ops.group_norm_act(h, 2, params[1], params[2], act="relu").permute(0, 2, 3, 1)
    y = ops.linear_act(h.reshape(12, 72), params[3], params[4], act="silu", res=target.cuda())
    got = (y.float() - 1).square().mean()
    # y is within some roundings of bf16 of its values, which lie below 8
    assert abs(got.item() - loss.item()) <= 8 * 8 * 2.0 ** -8 * loss.sqrt().item()
    ops.adamw_step([p.detach() for p in params], torch.autograd.grad(got, params), *state, 2.0 ** -6,
                   weight_decay=0.0, seed=4)
    m = ops.adamw_dequantize(*state[:2])[0].cpu().split([math.prod(s) for s in sizes])
    for p, q, g, first in zip(wide, params, grads, m):
        sure = g.abs() > 0.25 * g.abs().max()
        assert sure.any()
        want = (p - 2.0 ** -6 * g.sign())[sure]
        # a step of bf16 for its rounding, and what the moments' eps leaves of lr
        _within(q.detach()[sure.cuda()], want.detach(), 2.0 ** -7 * want.detach().abs() + 1e-4 * 2.0 ** -6)
        assert (first.view(g.shape)[sure].sign() == g[sure].sign()).all()


def test_captured_and_eager_epochs_agree_where_gradients_are_large(monkeypatch):
    """16 samples summed in another order change a gradient by 16 * 24 u of what enters its sum.
    Where a first moment is over a tenth of its largest, that is at most 64 times the gradient, and
    a step changes by twice that share of lr; four steps."""
    from torch.utils.data import DataLoader, TensorDataset

    from murmura_amd.aggregation.fedavg import FedAvgAggregator
    from murmura_amd.core.node import Node
    from murmura_amd.core.optim import AdamWConfig
    from murmura_amd.models import SimpleMLP

    def train(graphs):
        if not graphs:
            monkeypatch.setenv("MURMURA_NO_GRAPHS", "1")
        torch.manual_seed(0)
        data = TensorDataset(_randn((16, 24), FP32, 9), torch.arange(16) % 4)
        loader = DataLoader(data, batch_size=16)
        node = Node(0, SimpleMLP(24, 64, 4, fused=True), loader, loader, FedAvgAggregator(),
                    torch.device("cuda"), dtype=FP32, optimizer=AdamWConfig())
        for _ in range(4):
            node.local_train(lr=1e-2)
        monkeypatch.delenv("MURMURA_NO_GRAPHS", raising=False)
        return node

    a, b = train(True), train(False)
    sure = a.optimizer.exp_avg.abs() > 0.1 * a.optimizer.exp_avg.abs().max()
    assert sure.sum() > 20
    assert (a.get_state() - b.get_state())[sure].abs().max() <= 4 * 2 * 1e-2 * 16 * 24 * U * 64


@pytest.mark.parametrize("n,c,h,groups,act", [(128, 256, 56, 32, "silu"), (37, 48, 61, 3, "gelu"), (2, 64, 200, 8, "relu")])
def test_group_norm_repeats_between_other_calls(n, c, h, groups, act):
    """The same bits each time, in whichever of the three forms: held, read twice, by chunks."""
    def state(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        images = [torch.randn(n, h, h, c, generator=g, device="cuda").to(BF16).permute(0, 3, 1, 2) for _ in range(2)]
        w, b = (torch.randn(c, generator=g, device="cuda").to(BF16) for _ in range(2))
        return [t.requires_grad_(True) for t in (images[0], w, b)], images[1]

    def run(leaves, dy):
        y = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], act=act)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    one, two = state(1), state(2)
    first = run(*one)
    for _ in range(3):
        run(*two)
        assert all(torch.equal(p, q) for p, q in zip(first, run(*one)))


@pytest.mark.parametrize("act", ["relu", "silu"])
def test_linear_repeats_between_other_calls(act):
    """Sums split over parts are joined in their order."""
    def run(seed, m, k, n):
        g = torch.Generator("cuda").manual_seed(seed)
        x, w, dy = (torch.randn(s, generator=g, device="cuda").to(BF16) for s in ((m, k), (n, k), (m, n)))
        b = torch.randn(n, generator=g, device="cuda")
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        y = ops.linear_act(*leaves, act=act)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    for sizes in ((64, 3136, 2048), (1000, 1001, 999), (2048, 2048, 2048), (5, 7000, 40)):
        first = run(1, *sizes)
        for _ in range(3):
            run(2, *sizes)
            assert all(torch.equal(p, q) for p, q in zip(first, run(1, *sizes)))
