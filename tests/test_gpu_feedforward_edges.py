"""GPU: values at the edges of the feed-forward operators' ranges, against 64-bit results."""
import pytest
import torch
from torch.autograd import forward_ad

from gsc_amd import ops
from tests.feedforward_bounds import U, close, gated_bounds, half, wide

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,D", [(5, 16), (40, 16), (300, 16), (40, 1032), (300, 1032), (8518, 16)])
def test_gated_linear_gradients_with_an_infinite_gate_weight(M, D, dtype):
    """sigmoid of an infinite gate is 0 or 1 and its derivative 0: the gradients of weight and bias are finite, and the rows
    of the last tile that are not there add nothing to them."""
    g = torch.Generator().manual_seed(M + D)
    F = 72
    x, w = _randn(g, M, D, dtype=dtype), _randn(g, 2 * F, D, dtype=dtype, scale=D ** -0.5)
    b, dh = _randn(g, 2 * F, dtype=dtype), _randn(g, M, F, dtype=dtype)
    x[:, 0] = torch.where(x[:, 0] == 0, torch.ones_like(x[:, 0]), x[:, 0])   # 0 inf is no number
    big = w.clone()                      # the same function to 64 bits, with finite values: the sigmoid is 0 or 1 there
    w[3, 0], w[F - 1, 0] = float("inf"), float("-inf")
    big[3, 0], big[F - 1, 0] = 1e30, -1e30
    assert (x[:, 0].abs() > 1e-20).all()
    leaves = [t.requires_grad_() for t in (w, b)]
    h = ops.gated_linear(x, w, b, activation="sigmoid")
    dw, db = torch.autograd.grad(h, leaves, dh)
    want = gated_bounds(x, big, b, dh, "sigmoid", dtype)
    rows = torch.ones(2 * F, dtype=torch.bool)
    rows[[3, F - 1]] = False             # bounds of these gates' own gradients grow with the weight: they are 0
    for name, got in (("dw", dw), ("db", db)):
        v, tol = want[name]
        assert not got[~rows.cuda()].any()
        up = rows.clone()
        up[[F + 3, 2 * F - 1]] = False   # exact a = 0, 1: their bounds are those of the sum alone
        close(name, got[up.cuda()], v[up], tol[up], dtype)
        sums = (M + 8) * 2.0 ** -23 * (dh.detach().cpu().double().abs().t() @ (x.cpu().double().abs() if name == "dw" else
                                                                             torch.ones(M, 1, dtype=torch.float64)))
        a = ((x[:, :1].cpu().double() > 0) == torch.tensor([True, False])).double()          # of gates 3 and F - 1
        exact = (dh[:, [3, F - 1]].cpu().double() * a).t() @ (x.cpu().double() if name == "dw" else
                                                              torch.ones(M, 1, dtype=torch.float64))
        sel = [F + 3, 2 * F - 1]
        close(name, got[sel].reshape(exact.shape), exact, sums[[3, F - 1]], dtype)


@pytest.mark.parametrize("rows", [5, 40])
def test_gated_linear_casts_overlapping_rows(rows):
    """fp32 windows of one another's elements under autocast: the cast changes their strides (fewer rows than columns)."""
    g = torch.Generator().manual_seed(rows)
    t, w, dh = _randn(g, 80), _randn(g, 48, 24), _randn(g, rows, 24, dtype=BF16)
    windows = t.unfold(0, 24, 1)[:rows]
    out = []
    for x in (windows, windows.contiguous()):
        with torch.autocast("cuda", dtype=BF16):
            with torch.no_grad():
                first = ops.gated_linear(x, w)
            leaf = w.detach().clone().requires_grad_()
            h = ops.gated_linear(x, leaf)
        out.append((first, h.detach(), torch.autograd.grad(h, leaf, dh)[0]))
    assert all(torch.equal(a, b) for a, b in zip(*out))


NORM_WIDTHS = [1, 2, 7, 15, 30, 41, 320, 1003, 4095, 8192, 16384, 16395, 40000]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C", NORM_WIDTHS)
def test_layer_norm_rows_of_equal_values(C, dtype):
    """y is the bias, bit for bit, whatever the value and the length of the row; dx = (g - mean g) / sqrt(eps), dw = 0."""
    g = torch.Generator().manual_seed(C)
    values = torch.tensor([7.0, 300.0, 30000.0, 0.1, -1 / 3, 1e8, -1e-3, 0.0], dtype=dtype)
    x = values[:, None].repeat(1, C).cuda().requires_grad_()
    w, b = (_randn(g, C) + 1).requires_grad_(), _randn(g, C).requires_grad_()
    dy = _randn(g, len(values), C, dtype=dtype)
    y = ops.layer_norm(x, w, b)
    assert torch.equal(y.detach(), b.detach().to(dtype).expand_as(x))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    gw = wide(dy) * wide(w)
    r = 1e-5 ** -0.5
    want = r * (gw - gw.mean(-1, keepdim=True))
    # a sum of C terms, the mean's factor, eps in fp32, its root and the two products: C + 8 roundings of U
    tol = (C + 8) * U * r * (gw.abs() + gw.abs().mean(-1, keepdim=True))
    close("dx", dx, want, tol, dtype)
    assert not dw.any()
    close("db", db, wide(dy).sum(0), (len(values) + 1) * U * wide(dy).abs().sum(0), F32)


@pytest.mark.parametrize("C", [c for c in NORM_WIDTHS if c > 2])
@pytest.mark.parametrize("mean", [300.0, 30000.0, -1e6])
def test_layer_norm_rows_with_a_far_mean(C, mean):
    """The mean loses its own rounding and no more: U |mean|, not the roundings of a sum of C terms of its size."""
    g = torch.Generator().manual_seed(C)
    x, w = _randn(g, 9, C) * 3 + mean, _randn(g, C) + 1
    X, W = wide(x), wide(w)
    mu = X.mean(-1, keepdim=True)
    d = X - mu
    r = (d.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    # mean: its own rounding and C + 6 of the centred values, which the first estimate moves by at most (C + 2) U |mean|
    off = (C + 2) * U * abs(mean)
    emu = U * mu.abs() + (C + 6) * U * (d.abs().mean(-1, keepdim=True) + off)
    # squares: C + 8 roundings relative to the mean square about the first estimate, below twice the variance where off is
    # small and summed again where not; half of it in r.  The moved mean adds its square.
    er = (C + 8) * U + (emu * r).square()
    want = d * r * W
    close("y", ops.layer_norm(x, w), want, W.abs() * (r * emu + (d * r).abs() * (er + 4 * U)) + U * want.abs(), F32)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C", [7, 300, 16395])
def test_layer_norm_spread_below_the_mean_of_a_long_sum(C, dtype):
    """One value of a row differs by a step of its type: 1 / std is that of the values, not of the mean's roundings."""
    step = 2.0 ** (-7 if dtype == BF16 else -23)
    x = torch.full((3, C), 1.0, dtype=torch.float64)
    x *= torch.tensor([[30000.0], [1e6], [1.0]]).to(dtype).double()
    top = 2.0 ** x.log2().floor()
    x[:, C // 2] += step * top[:, C // 2]
    x = x.to(dtype).cuda().requires_grad_()
    X = wide(x)
    mu = X.mean(-1, keepdim=True)
    d = X - mu
    var = d.square().mean(-1, keepdim=True)
    r = (var + 1e-5).rsqrt()
    # the kernel's mean is the rounded one: its squares are about that, var + (its error)^2, at most U |mean|
    g = torch.Generator().manual_seed(C)
    dy = _randn(g, 3, C, dtype=dtype)
    (dx,) = torch.autograd.grad(ops.layer_norm(x), x, dy)
    m32 = mu.float().double()
    worst = []
    for m in (m32, torch.nextafter(mu.float(), torch.tensor(1e30)).double(), torch.nextafter(mu.float(), torch.tensor(0.0)).double()):
        e = X - m
        rr = (e.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        G, xh = wide(dy), e * rr
        want = rr * (G - G.mean(-1, keepdim=True) - xh * (G * xh).mean(-1, keepdim=True))
        tol = (2 * C + 24) * U * rr * (G.abs() + G.abs().mean(-1, keepdim=True) + xh.abs() * (G * xh).abs().mean(-1, keepdim=True))
        err = (dx.cpu().double() - want).abs() / (tol + half(dtype) * (want.abs() + tol))
        worst.append(err.amax(-1))
    # the mean in fp32 is one of the neighbours of the exact one
    assert (torch.stack(worst).amin(0) <= 1.0).all(), worst


def _calls(x, w, gw, gb):
    return {"layer_norm": (lambda **k: ops.layer_norm(**{"x": x, "weight": w, "bias": w, **k}), ("x", "weight", "bias")),
            "dropout": (lambda **k: ops.dropout(**{"x": x, "p": 0.1, "seed": 1, "residual": x, **k}), ("x", "residual")),
            "gated_linear": (lambda **k: ops.gated_linear(**{"x": x, "weight": gw, "bias": gb, **k}), ("x", "weight", "bias"))}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", ["layer_norm", "dropout", "gated_linear"])
def test_forward_mode_is_refused(name, grad):
    """A tangent on any input is refused, with and without gradients; inputs without one pass at an open dual level."""
    g = torch.Generator().manual_seed(1)
    tensors = _randn(g, 5, 8), _randn(g, 8), _randn(g, 12, 8), _randn(g, 12)
    call, names = _calls(*tensors)[name]
    like = dict(zip(("x", "weight", "bias"), (tensors[0], *(tensors[2:] if name == "gated_linear" else (tensors[1],) * 2))),
                residual=tensors[0])
    want = call()
    with forward_ad.dual_level():
        assert torch.equal(call(), want)
        for k in names:
            dual = forward_ad.make_dual(like[k].clone().requires_grad_(grad), torch.ones_like(like[k]))
            with pytest.raises(NotImplementedError, match=name):
                call(**{k: dual})


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("name", ["layer_norm", "dropout", "gated_linear"])
def test_tracing_without_gradients_is_refused(name):
    g = torch.Generator().manual_seed(2)
    x = _randn(g, 5, 8)
    call, _ = _calls(x, _randn(g, 8), _randn(g, 12, 8), _randn(g, 12))[name]
    with pytest.raises(RuntimeError, match=f"{name}: cannot be traced"):
        torch.jit.trace(lambda t: call(x=t), x, check_trace=False)


def _activation64(g, act):
    """act(g), act'(g) in 64 bits, and the sum of the derivative's terms (what its roundings are relative to)."""
    s = torch.sigmoid(g)
    if act == "gelu":
        phi, e = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5), torch.exp(-0.5 * g * g) * (0.5 / torch.pi) ** 0.5
        return g * phi, phi + g * e, phi + (g * e).abs()
    c = torch.sigmoid(-g)
    # 1 - s, of a rounded s, is off by U: two roundings relative to s itself
    return (g * s, s * (1 + g * c), s * (1 + g.abs() * (c + 1))) if act == "silu" else (s, s * c, s * (c + 1))


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [30, 4001])
def test_activations_are_right_relative_to_their_own_size(rows, dtype, act):
    """Values and derivatives over g in -12 .. 12, the small ones of the negative side included (up projection 1)."""
    g = torch.linspace(-12, 12, rows).to(dtype).cuda()
    x = torch.zeros(rows, 8, device="cuda", dtype=dtype)
    x[:, 0] = g
    w, b = torch.zeros(8, 8, device="cuda", dtype=dtype), torch.zeros(8, device="cuda")
    w[:4, 0] = 1.0      # four gates of x[:, 0]
    b[4:] = 1.0
    x.requires_grad_()
    h = ops.gated_linear(x, w, b, activation=act)
    dh = torch.zeros_like(h)
    dh[:, 1] = 1.0
    (dx,) = torch.autograd.grad(h, x, dh)
    a, d, size = _activation64(wide(g), act)
    # exponent: rounding of g^2 / 2 and, in bf16, of its product with log2 e, g^2 U together (|g| U of the others, which is
    # less than g^2 U + U); exponential, reciprocal and the operations around them 12 U; the polynomial 6.2e-8 < 2 U and its
    # roundings 3 U
    rel = (wide(g).square() + 18) * U
    for k in range(4):
        close("h", h[:, k], a, rel * a.abs(), dtype)
    # dg is a matrix operand: rounded to the type once more
    tol = rel * size
    close("dx", dx[:, 0], d, tol + (half(dtype) * (d.abs() + tol) if dtype == BF16 else 0), dtype)


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("M", [4, 200])
def test_fp32_activations_of_huge_gates(M, act):
    """Gates of 1e29: the activation is 0 or the gate itself (sigmoid: 0 or 1), their product with the up projection 0,
    infinite or the projection."""
    g = torch.Generator().manual_seed(M)
    x, w = torch.zeros(M, 100, device="cuda"), _randn(g, 120, 100, scale=0.1)
    x[:, 0] = 3e30 * torch.where(torch.arange(M, device="cuda") % 2 == 0, 1.0, -1.0)
    h = ops.gated_linear(x, w, activation=act)
    gate, up = (wide(x) @ wide(w).t()).chunk(2, 1)
    on = gate > 0
    if act == "sigmoid":
        close("h", h, torch.where(on, up, 0.0), 4 * U * up.abs(), F32)
    else:
        assert torch.equal(h.cpu(), torch.where(on, torch.inf * up.sign(), 0.0).float())


@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_fp32_small_values_of_the_sigmoid(act):
    """Gates down to -80: the exponential's relative error does not grow with its argument."""
    g = torch.linspace(-80, 0, 4001, device="cuda")
    x, w = torch.zeros(4001, 8, device="cuda"), torch.zeros(2, 8, device="cuda")
    x[:, 0], w[0, 0] = g, 1.0
    h = ops.gated_linear(x, w, torch.tensor([0.0, 1.0], device="cuda"), activation=act)
    a = _activation64(wide(g), act)[0]
    close("h", h[:, 0], a, 8 * U * a.abs(), F32)   # exponential, sum, quotient, two products: 8 roundings at most


def test_capture_beside_a_graph_of_another_operator():
    """A living graph of the same leaf is noticed whatever operator made it: refused where it belongs to another stream,
    not where it is part of the capture itself."""
    g = torch.Generator().manual_seed(3)
    x, nw, gw = _randn(g, 20, 32), (_randn(g, 32) + 1).requires_grad_(), _randn(g, 16, 32).requires_grad_()
    calls = {"norm": (lambda: ops.layer_norm(x, nw), nw), "gated": (lambda: ops.gated_linear(x, gw), gw),
             "dropout": (lambda: ops.dropout(gw, 0.5, 1, 1), gw)}
    for call, leaf in calls.values():
        alive = leaf * 2
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        assert torch.equal(torch.autograd.grad(alive.sum(), leaf)[0], torch.full_like(leaf, 2.0))
        del alive

        def both():
            twice = leaf * 2               # holds the leaf's node before the operator sees it
            y = call()
            return torch.autograd.grad((twice.sum(), y), leaf, (None, torch.ones_like(y)))[0]

        want = both()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = both()
        for _ in range(3):
            got.zero_()
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            assert torch.equal(both(), want)


@pytest.mark.parametrize("B", [100, 25600])
def test_graphed_updates_of_the_trained_batches(B):
    """The batches of one and of 256 environments: replays equal eager updates, library reductions in the graph included."""
    from tests.test_gpu_feedforward_learner import test_graphed_updates_equal_eager_ones
    test_graphed_updates_equal_eager_ones(B)
