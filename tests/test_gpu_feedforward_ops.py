"""GPU: layer norm, counter-based dropout and the gated linear layer against 64-bit results with counted error bounds."""
import pytest
import torch

from gsc_amd import ops
from tests.feedforward_bounds import U, close, gated_bounds, half, layer_norm_bounds, wide

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _gen(*key):
    return torch.Generator().manual_seed(sum((i + 1) * 7919 * (hash(k) % 1009 if isinstance(k, str) else int(k))
                                             for i, k in enumerate(key)) % (1 << 31))


def _randn(g, *shape, dtype=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).cuda()


# ---------------------------------------------------------------------------------------------------------------
# layer norm

NORM_SHAPES = [(1, 1), (5, 2), (1, 7), (300, 22), (3, 64), (64, 128), (5, 255), (70, 256), (17, 257), (9, 512), (2, 1003),
               (6, 1024), (3, 2048), (5, 4095), (3, 4096), (2, 8192), (2, 8200), (3, 16384), (2, 16385), (1, 40000),
               (2051, 40)]


def _norm_check(x, w, b, dy, eps=1e-5):
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = ops.layer_norm(x, w, b, eps)
    with torch.no_grad():
        assert torch.equal(y, ops.layer_norm(x, w, b, eps))
    grads = dict(zip([n for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None],
                     torch.autograd.grad(y, leaves, dy)))
    want = layer_norm_bounds(x.reshape(-1, x.shape[-1]), w, b, dy.reshape(-1, x.shape[-1]), eps)
    close("y", y.reshape(-1, x.shape[-1]), *want["y"], x.dtype)
    close("dx", grads["dx"].reshape(-1, x.shape[-1]), *want["dx"], x.dtype)
    if w is not None:
        close("dw", grads["dw"], *want["dw"], w.dtype)
    if b is not None:
        close("db", grads["db"], *want["db"], b.dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_layer_norm(shape, dtype):
    g = _gen(*shape)
    x = _randn(g, *shape, dtype=dtype, shift=0.5)
    w, b = _randn(g, shape[1], scale=0.2, shift=1.0), _randn(g, shape[1], scale=0.2)
    _norm_check(x, w, b, _randn(g, *shape, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("wt,bt", [(None, None), (BF16, None), (None, F32), (BF16, BF16), (F32, BF16)])
def test_layer_norm_parameter_types(dtype, wt, bt):
    g = _gen(3)
    x = _randn(g, 33, 96, dtype=dtype)
    w = _randn(g, 96, dtype=wt, shift=1.0) if wt else None
    b = _randn(g, 96, dtype=bt) if bt else None
    _norm_check(x, w, b, _randn(g, 33, 96, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("wt", [BF16, F32])
@pytest.mark.parametrize("C", [*range(1, 18), 29, 509, 1021, 8187, 16395])
def test_layer_norm_rows_between_nan(C, dtype, wt):
    """Rows and parameters that start and end anywhere, with NaN in front of and behind each."""
    g = _gen(49, C)

    def inside(*shape, t, **kw):
        out = torch.full((*shape[:-1], C + 11), float("nan"), device="cuda", dtype=t)
        out[..., 5:5 + C] = _randn(g, *shape, dtype=t, **kw)
        return out[..., 5:5 + C]

    x, dy = inside(6, C, t=dtype, shift=0.5), inside(6, C, t=dtype)
    _norm_check(x, inside(C, t=wt, scale=0.2, shift=1.0), inside(C, t=wt, scale=0.2), dy)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("how", ["slice", "odd_slice", "transposed", "three_d", "one_d", "grad_expanded", "x_expanded",
                                 "grad_slice"])
def test_layer_norm_strides(dtype, how):
    """Row views, copies where no row view exists, broadcast inputs and gradients, rows off any vector alignment."""
    g = _gen(4)
    C = 200
    base = _randn(g, 21, 512, dtype=dtype)
    x = {"slice": lambda: base[:, 8:8 + C], "odd_slice": lambda: base[:, 3:3 + C], "transposed": lambda: base[:, :C].t(),
         "three_d": lambda: base[:20, :C].reshape(4, 5, C), "one_d": lambda: base[0, :C],
         "x_expanded": lambda: base[:1, :C].expand(21, C)}.get(how, lambda: base[:, :C])()
    dy = _randn(g, *x.shape, dtype=dtype)
    if how == "grad_expanded":
        dy = dy[:1].expand_as(dy)
    if how == "grad_slice":
        dy = _randn(g, 21, 333, dtype=dtype)[:, 5:5 + C]
    C = x.shape[-1]
    _norm_check(x.detach(), _randn(g, C, shift=1.0), _randn(g, C), dy)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layer_norm_hard_rows(dtype):
    """Constant rows give the bias, far means lose what their size costs and no more, non-finite rows stay alone."""
    g = _gen(5)
    C = 320
    w, b = _randn(g, C, shift=1.0), _randn(g, C)
    x = _randn(g, 6, C, dtype=dtype)
    x[1] = 7.0
    x[2] = 0.0
    x[3] = x[3] * 0.01 + 300.0
    dy = _randn(g, 6, C, dtype=dtype)
    _norm_check(x.clone(), w, b, dy)
    ref = ops.layer_norm(x, w.detach(), b.detach())
    assert torch.equal(ref[1], b.detach().to(dtype))
    x[4, 17] = float("inf")
    x[5, 3] = float("nan")
    out = ops.layer_norm(x, w.detach(), b.detach())
    assert torch.equal(out[:4], ref[:4]) and out[4:].isnan().all()


@pytest.mark.parametrize("rows", [0, 1])
def test_layer_norm_no_rows(rows):
    x = torch.randn(rows, 5, 48, device="cuda")[:, :0 if rows else 5].requires_grad_(True)
    w = torch.ones(48, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert y.shape == x.shape and dx.shape == x.shape and not dw.any()


def test_layer_norm_gradients_of_some():
    """Only what is asked for is computed, and it equals what is computed together."""
    g = _gen(6)
    x, w, b, dy = _randn(g, 40, 72), _randn(g, 72, shift=1.0), _randn(g, 72), _randn(g, 40, 72)
    full = torch.autograd.grad(ops.layer_norm(x.requires_grad_(), w.requires_grad_(), b.requires_grad_()), (x, w, b), dy)
    for i in range(3):
        ts = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(ops.layer_norm(*ts), ts[i], dy)[0], full[i])


def test_layer_norm_many_rows_reproducible():
    g = _gen(7)
    x, w, b = _randn(g, 25600, 64, dtype=BF16), _randn(g, 64, shift=1.0), _randn(g, 64)
    dy = _randn(g, 25600, 64, dtype=BF16)
    _norm_check(x, w, b, dy)
    a = torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), dy)
    c = torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip(a, c))


# ---------------------------------------------------------------------------------------------------------------
# dropout

def _drop_check(x, res, p, seed, offset, dy, **kw):
    leaves = [t.requires_grad_(True) for t in (x, res) if t is not None]
    y = ops.dropout(x, p, seed, kw.get("at", offset), residual=res)
    grads = torch.autograd.grad(y, leaves, dy)
    keep = ops.dropout_mask(x.shape, p, seed, offset)
    scaled = torch.where(keep, wide(x) / (1 - p), 0.0)
    want = scaled + (wide(res) if res is not None else 0.0)
    close("y", y, want, 2 * U * scaled.abs() + U * want.abs() * (res is not None), x.dtype)
    dx = torch.where(keep, wide(dy) / (1 - p), 0.0)
    close("dx", grads[0], dx, 2 * U * dx.abs(), x.dtype)
    assert torch.equal(grads[0].cpu()[~keep], torch.zeros(int((~keep).sum()), dtype=x.dtype))
    if res is not None:
        assert torch.equal(grads[1], dy)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9, 1), (100, 64), (3, 5, 17), (513, 31), (2048, 64), (1000, 333)])
def test_dropout(shape, residual, dtype):
    g = _gen(11, *shape)
    x, dy = _randn(g, *shape, dtype=dtype), _randn(g, *shape, dtype=dtype)
    _drop_check(x, _randn(g, *shape, dtype=dtype) if residual else None, 0.3, 12345, 6, dy)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -32, 1e-6, 0.5, 1 / 3, 0.999, 1 - 2.0 ** -40])
@pytest.mark.parametrize("seed,offset", [(0, 0), ((1 << 64) - 1, (1 << 63) - 1), (1 << 40, 1 << 35)])
def test_dropout_probabilities_and_counters(p, seed, offset):
    g = _gen(12)
    _drop_check(_randn(g, 40, 50), None, p, seed, offset, _randn(g, 40, 50))


def test_dropout_decides_ties_by_the_second_block():
    """Thresholds inside the 16-bit step of chosen elements: their upper halves equal the threshold's, so the lower
    halves decide, and a threshold one above or at the uniform drops or keeps that element."""
    n, seed, offset = 4096, 77, 5
    from gsc_amd.ops.philox_dropout import _philox
    halves = lambda w: torch.from_numpy(w.astype("int64")).view(-1, 4, 1).bitwise_right_shift(
        torch.tensor([0, 16])).bitwise_and(0xFFFF).reshape(-1)
    u = halves(_philox(n // 8, seed, offset)) * 65536 + halves(_philox(n // 8, seed, offset | 1 << 63))
    x = torch.ones(n, device="cuda")
    for i in (0, 9, 1234, 4095):
        for thr, kept in ((int(u[i]), True), (int(u[i]) + 1, False)):
            y = ops.dropout(x, thr * 2.0 ** -32, seed, offset).cpu()
            assert bool(y[i] != 0) is kept
            assert torch.equal(y != 0, u >= thr)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("how", ["slice", "transposed", "unaligned", "expanded"])
def test_dropout_strides(dtype, how):
    """The mask goes by the logical index, whatever the strides."""
    g = _gen(13)
    base = _randn(g, 65, 130, dtype=dtype)
    mk = {"slice": lambda t: t[1:, 3:67], "transposed": lambda t: t[:64, :64].t(), "expanded": lambda t: t[:1, :64].expand(64, 64),
          "unaligned": lambda t: t.reshape(-1)[1:1 + 64 * 64].view(64, 64)}[how]
    x, dy, res = mk(base).detach(), mk(_randn(g, 65, 130, dtype=dtype)), mk(_randn(g, 65, 130, dtype=dtype)).detach()
    _drop_check(x, None, 0.4, 3, 1, dy)
    _drop_check(x.detach(), res, 0.4, 3, 1, dy)


def test_dropout_drops_nonfinite_values_and_rate():
    x = torch.full((1 << 20,), float("nan"), device="cuda")
    y = ops.dropout(x, 0.25, 5, 9)
    keep = ops.dropout_mask(x.shape, 0.25, 5, 9)
    assert torch.equal(y.isnan().cpu(), keep) and not y[~keep.cuda()].any()
    # 2^20 draws of probability 3/4: six standard deviations are 6 sqrt(n p (1 - p)) = 2661
    assert abs(int(keep.sum()) - 0.75 * (1 << 20)) < 2661


def test_dropout_masks_differ_by_seed_and_offset():
    x = torch.ones(1 << 16, device="cuda")
    a, b, c = (ops.dropout(x, 0.5, s, o) != 0 for s, o in ((1, 1), (2, 1), (1, 2)))
    for p, q in ((a, b), (a, c), (b, c)):   # agreement of independent fair bits: 2^15 +- 6 * 128
        assert abs(int((p == q).sum()) - (1 << 15)) < 768
    assert torch.equal(a, ops.dropout(x, 0.5, 1, 1) != 0)


def test_dropout_offset_tensor():
    """A device offset is read when the kernel runs, and the backward pass keeps the value its forward read."""
    g = _gen(14)
    at = torch.tensor([41], device="cuda")
    x, dy = _randn(g, 30, 70), _randn(g, 30, 70)
    _drop_check(x, None, 0.2, 8, 41, dy, at=at)
    y = ops.dropout(x, 0.2, 8, at)
    at.add_(1)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx != 0, y != 0)
    assert torch.equal(ops.dropout(x, 0.2, 8, at), ops.dropout(x, 0.2, 8, 42))


def test_dropout_beyond_32_bit_elements():
    """Groups are counted in 64 bits: the end of a tensor of more than 2^32 elements."""
    n = (1 << 32) + 24
    x = torch.ones(n, device="cuda", dtype=BF16)
    y = ops.dropout(x, 0.5, 21, 3)
    from gsc_amd.ops.philox_dropout import _philox  # noqa: F401
    head = ops.dropout_mask((64,), 0.5, 21, 3)
    assert torch.equal((y[:64] != 0).cpu(), head)
    # the last 24 elements are groups 2^29 .. 2^29 + 2: their blocks directly
    import numpy as np
    g0 = (1 << 29)
    words = _blocks_at(np.arange(g0, g0 + 3, dtype=np.uint64), 21, 3)
    hi = np.stack((words & 0xFFFF, words >> 16), -1).reshape(-1)
    assert (hi != 0x8000).all()   # no tie at p = 1/2: the upper halves decide
    assert torch.equal((y[-24:] != 0).cpu(), torch.from_numpy(hi >= 0x8000))


def _blocks_at(groups, seed, offset):
    import numpy as np
    m, s = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [groups & m, groups >> s, np.full_like(groups, offset & 0xFFFFFFFF), np.full_like(groups, offset >> 32)]
    for r in range(10):
        k0, k1 = np.uint64((seed + r * 0x9E3779B9) & 0xFFFFFFFF), np.uint64(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> s) ^ c[1] ^ k0, p1 & m, (p0 >> s) ^ c[3] ^ k1, p0 & m]
    return np.stack(c, 1).astype(np.uint32)


# ---------------------------------------------------------------------------------------------------------------
# gated linear layer

GATED_SHAPES = [(1, 1, 1), (1, 256, 1024), (2, 8, 5), (3, 100, 33), (8, 512, 96), (16, 64, 64), (33, 72, 40), (64, 22, 256),
                (65, 257, 129), (100, 64, 256), (130, 96, 200), (257, 264, 136), (300, 31, 77), (600, 320, 512),
                (1100, 128, 640), (4200, 72, 2101), (4200, 4104, 72), (100, 4104, 2104), (40, 1032, 72),
                (200, 1100, 130), (2200, 1024, 1100), (90, 128, 64), (8518, 16, 1024), (8518, 1032, 1020),
                (33, 4096, 70), (130, 2050, 129), (700, 1500, 60)]


def _gated_check(x, w, b, dh, act, op, w_used=None):
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    h = ops.gated_linear(x, w, b, activation=act)
    with torch.no_grad():
        assert torch.equal(h, ops.gated_linear(x, w, b, activation=act))
    grads = dict(zip([n for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None],
                     torch.autograd.grad(h, leaves, dh)))
    D, F = x.shape[-1], h.shape[-1]
    want = gated_bounds(x.reshape(-1, D).to(op), (w if w_used is None else w_used).to(op), b,
                        dh.reshape(-1, F).to(op), act, op)
    close("h", h.reshape(-1, F), *want["h"], op)
    close("dx", grads["dx"].reshape(-1, D), *want["dx"], x.dtype)
    close("dw", grads["dw"], *want["dw"], w.dtype)
    if b is not None:
        close("db", grads["db"], *want["db"], b.dtype)


def _gated_inputs(g, M, D, F, dtype):
    return (_randn(g, M, D, dtype=dtype), _randn(g, 2 * F, D, dtype=dtype, scale=D ** -0.5),
            _randn(g, 2 * F, dtype=dtype, scale=0.5), _randn(g, M, F, dtype=dtype))


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", GATED_SHAPES)
def test_gated_linear(shape, dtype, act):
    x, w, b, dh = _gated_inputs(_gen(21, *shape), *shape, dtype)
    _gated_check(x, w, b, dh, act, dtype)


@pytest.mark.parametrize("how", ["x_slice", "x_odd", "w_slice", "w_odd", "w_transposed", "three_d", "one_d", "dh_expanded",
                                 "dh_slice", "no_bias", "fp32_bias", "f_odd"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gated_linear_layouts(dtype, how):
    g = _gen(22)
    M, D, F = 70, 96, 80 if how != "f_odd" else 77
    x, w, b, dh = _gated_inputs(g, M, D, F, dtype)
    if how == "x_slice":
        x = _randn(g, M, 200, dtype=dtype)[:, 16:16 + D].detach()
    elif how == "x_odd":
        x = _randn(g, M, 201, dtype=dtype)[:, 3:3 + D].detach()
    elif how == "w_slice":
        w = _randn(g, 2 * F, 200, dtype=dtype, scale=0.1)[:, 8:8 + D].detach()
    elif how == "w_odd":
        w = _randn(g, 2 * F, 201, dtype=dtype, scale=0.1)[:, 5:5 + D].detach()
    elif how == "w_transposed":
        w = _randn(g, D, 2 * F, dtype=dtype, scale=0.1).t().detach()
    elif how == "three_d":
        x, dh = x.view(2, 35, D), dh.view(2, 35, F)
    elif how == "one_d":
        x, dh = x[0].clone(), dh[0].clone()
    elif how == "dh_expanded":
        dh = dh[:1].expand(M, F)
    elif how == "dh_slice":
        dh = _randn(g, M, F + 9, dtype=dtype)[:, 3:3 + F]
    elif how == "no_bias":
        b = None
    elif how == "fp32_bias":
        b = b.float()
    _gated_check(x, w, b, dh, "silu", dtype)


def test_gated_linear_masters_and_autocast():
    """fp32 masters beside bf16 activations: the operand is the shadow (or a cast), the gradients come back in fp32."""
    g = _gen(23)
    x, w, b, dh = _gated_inputs(g, 90, 64, 48, F32)
    w16 = (w + 0.01).bfloat16()                      # a shadow that differs, to see which one is used
    _gated_check(x.bfloat16().detach(), w.detach(), b.detach(), dh.bfloat16(), "gelu", BF16)
    shadowed = w.detach().clone()
    shadowed._bf16 = w16
    _gated_check(x.bfloat16().detach(), shadowed, b.detach(), dh.bfloat16(), "gelu", BF16, w_used=w16)
    with torch.autocast("cuda", dtype=BF16):
        _gated_check(x.detach(), w.detach(), b.detach(), dh.bfloat16(), "silu", BF16)


def test_gated_linear_no_rows():
    x = torch.empty(0, 24, device="cuda", requires_grad=True)
    w = torch.randn(20, 24, device="cuda", requires_grad=True)
    h = ops.gated_linear(x, w)
    dx, dw = torch.autograd.grad(h, (x, w), torch.ones_like(h))
    assert h.shape == (0, 10) and dx.shape == (0, 24) and dw.shape == w.shape and not dw.any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [4, 200])
def test_gated_linear_nonfinite_values_stay_in_their_row(M, dtype):
    g = _gen(24)
    x, w, b, _ = _gated_inputs(g, M, 100, 60, dtype)
    ref = ops.gated_linear(x, w, b)
    x[2, 99] = float("nan")
    out = ops.gated_linear(x, w, b)
    rest = torch.arange(M) != 2
    assert out[2].isnan().all() and torch.equal(out[rest.cuda()], ref[rest.cuda()])
    far = torch.zeros_like(x)
    far[:, 0] = 3e4 if dtype == BF16 else 3e30       # g and u of both signs, far in the tails of every activation
    for act in ("silu", "gelu", "sigmoid"):
        y = ops.gated_linear(far, w, b, activation=act)
        want = gated_bounds(far, w, b, None, act, dtype)["h"][0]
        if dtype == BF16:
            assert y.isfinite().all() and (y.cpu().double() - want).abs().max() <= 0.02 * want.abs().max()


def test_gated_linear_reproducible_and_partial_gradients():
    g = _gen(25)
    x, w, b, dh = _gated_inputs(g, 5000, 64, 64, BF16)
    full = torch.autograd.grad(ops.gated_linear(x.requires_grad_(), w.requires_grad_(), b.requires_grad_()), (x, w, b), dh)
    again = torch.autograd.grad(ops.gated_linear(x, w, b), (x, w, b), dh)
    assert all(torch.equal(p, q) for p, q in zip(full, again))
    for i in range(3):
        ts = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(ops.gated_linear(*ts), ts[i], dh)[0], full[i])


# ---------------------------------------------------------------------------------------------------------------
# together, on streams, in graphs

def _block(x, p, seed, at, train=True):
    n = ops.layer_norm(x, p["nw"], p["nb"])
    h = ops.gated_linear(n, p["w"], p["b"])
    d = torch.nn.functional.linear(h, p["wd"].to(h.dtype))
    return ops.dropout(d, 0.2, seed, at, residual=x) if train else d + x


def _block_params(g, D, F, dtype):
    return {"nw": _randn(g, D, shift=1.0, scale=0.1), "nb": _randn(g, D, scale=0.1),
            "w": _randn(g, 2 * F, D, dtype=dtype, scale=D ** -0.5), "b": _randn(g, 2 * F, scale=0.1),
            "wd": _randn(g, D, F, dtype=dtype, scale=F ** -0.5)}


def test_block_gradients_against_formula_and_differences():
    """The operators as one residual block in fp32: every gradient against autograd of the 64-bit references, and a
    directional derivative against central differences of the 64-bit block."""
    g = _gen(31)
    D, F, M = 40, 72, 50
    p = _block_params(g, D, F, F32)
    x, dy = _randn(g, M, D), _randn(g, M, D)
    names = list(p)
    for t in (x, *p.values()):
        t.requires_grad_(True)
    y = _block(x, p, 17, 4)
    grads = torch.autograd.grad(y, [x, *p.values()], dy)

    keep = ops.dropout_mask((M, D), 0.2, 17, 4)

    def block64(x, q):
        n = ops.layer_norm_reference(x, q["nw"], q["nb"])
        h = ops.gated_linear_reference(n, q["w"], q["b"])
        return torch.where(keep, h @ q["wd"].t() / 0.8, 0.0) + x

    x64, q64 = wide(x).requires_grad_(), {k: wide(v).requires_grad_() for k, v in p.items()}
    y64 = block64(x64, q64)
    want = torch.autograd.grad(y64, [x64, *q64.values()], wide(dy))
    # about D + F + 20 roundings of U along each path, magnified by the block's gains (below 30 for these inputs)
    tol = 30 * (D + F + 20) * U
    for n, a, b in zip(["x", *names], grads, want):
        assert (a.cpu().double() - b).norm() <= tol * b.norm(), n
    assert (y.cpu().double() - y64).norm() <= tol * y64.norm()
    with torch.no_grad():
        v = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (x64, *q64.values())]
        step = 1e-5

        def shifted(s):
            return (block64(x64 + s * v[0], {k: t + s * d for (k, t), d in zip(q64.items(), v[1:])}) * wide(dy)).sum()

        diff = (shifted(step) - shifted(-step)) / (2 * step)
        got = sum((a.cpu().double() * d).sum() for a, d in zip(grads, v))
        # the differences' own error: step^2 of third derivatives (below 1e3 of the scale) -> 1e-7, plus tol
        scale = sum((b.norm() * d.norm()).item() for b, d in zip(want, v))
        assert abs(got - diff) <= (tol + 1e-7) * scale


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_block_on_another_stream(dtype):
    g = _gen(32)
    p, x = _block_params(g, 64, 128, dtype), _randn(g, 300, 64, dtype=dtype)
    leaves = [t.requires_grad_(True) for t in (x, *p.values())]
    dy = _randn(g, 300, 64, dtype=dtype)
    want = torch.autograd.grad(_block(x, p, 1, 2), leaves, dy)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = torch.autograd.grad(_block(x, p, 1, 2), leaves, dy)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_block_captured_and_replayed():
    """Forward and backward captured in one HIP graph: every replay draws the next mask and equals the eager pass of the
    same offset, with eager work between the replays.  Two graphs of the same call do not share anything."""
    g = _gen(33)
    p, x = _block_params(g, 64, 96, BF16), _randn(g, 500, 64, dtype=BF16)
    leaves = [t.requires_grad_(True) for t in (x, *p.values())]
    dy = _randn(g, 500, 64, dtype=BF16)
    at = torch.zeros(1, device="cuda", dtype=torch.int64)

    def passes(offset):
        y = _block(x, p, 9, offset)
        return (y, *torch.autograd.grad(y, leaves, dy))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            passes(at)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            at.add_(1)
            out = passes(at)
        graphs.append((gr, out))
    at.zero_()
    for k in range(1, 7):
        gr, out = graphs[k % 2]
        gr.replay()
        got = [t.clone() for t in out]
        want = passes(k)
        torch.cuda.synchronize()
        assert int(at) == k
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_capture_refused_while_an_eager_graph_of_the_leaves_lives():
    """The gradient node of a leaf belongs to the stream of the graph that holds it: a captured backward pass through it
    would end the process, so the captured call is refused, for each operator, and works once that graph is gone."""
    g = _gen(34)
    x, w, gw = _randn(g, 20, 32), _randn(g, 32, shift=1.0).requires_grad_(), _randn(g, 16, 32).requires_grad_()
    calls = {"norm": (lambda: ops.layer_norm(x, w), w), "gated": (lambda: ops.gated_linear(x, gw), gw),
             "dropout": (lambda: ops.dropout(gw, 0.5, 1, 1), gw)}
    for call, leaf in calls.values():
        alive = call()
        gr = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(gr):
                call()
        want = torch.autograd.grad(alive, leaf, torch.ones_like(alive))[0]
        del alive, gr
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = call()
            (got,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
        gr.replay()
        assert torch.equal(got, want)
        del y, got, gr


def _each(g):
    """A call of each operator on fresh leaves, and the leaves."""
    x, w, gw = (_randn(g, 20, 32).requires_grad_(), _randn(g, 32, shift=1.0).requires_grad_(),
                _randn(g, 16, 32).requires_grad_())
    return [(lambda: ops.layer_norm(x, w), (x, w)), (lambda: ops.dropout(x, 0.5, 3, 1), (x,)),
            (lambda: ops.gated_linear(x, gw), (x, gw))]


def test_graph_kept_for_a_second_backward_pass():
    for call, leaves in _each(_gen(41)):
        y = call()
        dy = torch.ones_like(y)
        first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, leaves, dy)))


def test_second_derivatives_are_refused():
    """A gradient taken with create_graph is right, and differentiating it again raises instead of giving zeros."""
    for call, leaves in _each(_gen(42)):
        y = call()
        plain = torch.autograd.grad(y, leaves, torch.ones_like(y), retain_graph=True)
        dy = torch.ones_like(y).requires_grad_()
        grads = torch.autograd.grad(y, leaves, dy, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, grads))
        with pytest.raises(RuntimeError, match="once_differentiable"):
            grads[0].sum().backward()


def test_inputs_changed_before_the_backward_pass_are_noticed():
    g = _gen(43)
    x, w = _randn(g, 20, 32), _randn(g, 32, shift=1.0).requires_grad_()
    gw = _randn(g, 16, 32).requires_grad_()
    for call, leaf in ((lambda: ops.layer_norm(x, w), w), (lambda: ops.gated_linear(x, gw), gw)):
        y = call()
        x.add_(1.0)
        with pytest.raises(RuntimeError, match="inplace"):
            torch.autograd.grad(y, leaf, torch.ones_like(y))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [31, 1024])
def test_saved_tensors_moved_to_the_host_or_recomputed(D, dtype):
    """The gradients are those of a plain call, bit for bit, where a hook moves what a forward pass saved or the forward
    pass runs again before the backward one."""
    from torch.utils.checkpoint import checkpoint
    g = _gen(45, D)
    x, dy = _randn(g, 60, 2 * D, dtype=dtype)[:, :D], _randn(g, 60, 24, dtype=dtype)
    w, b = _randn(g, D, shift=1.0), _randn(g, D)
    gw, gb = _randn(g, 48, D, dtype=dtype, scale=D ** -0.5), _randn(g, 48, dtype=dtype)

    def block(x, w, b, gw, gb):
        return ops.dropout(ops.gated_linear(ops.layer_norm(x, w, b), gw, gb), 0.3, 5)

    def call(run):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, gw, gb)]
        y = run(leaves)
        spoil = torch.full((1 << 16,), float("nan"), device="cuda")   # reuses what the call freed
        del spoil
        return torch.autograd.grad(y, leaves, dy)

    def on_host(leaves):
        with torch.autograd.graph.save_on_cpu():
            return block(*leaves)

    plain = call(lambda leaves: block(*leaves))
    for run in (on_host, lambda leaves: checkpoint(block, *leaves, use_reentrant=False, preserve_rng_state=False)):
        assert all(torch.equal(a, c) for a, c in zip(plain, call(run)))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gated_linear_kept_products_equal_recomputed_ones(dtype):
    """On both sides of the widths from which the forward pass keeps its products: the same bounds hold, and a wider
    operand padded with zeros gives the same gradients as the narrow one."""
    g = _gen(44)
    D = 1016 if dtype == BF16 else 120
    x, w, b, dh = _gated_inputs(g, 150, D, 72, dtype)
    pad = lambda t: torch.cat([t, torch.zeros(t.shape[0], 8, device="cuda", dtype=t.dtype)], 1)
    out = []
    for xx, ww in ((x, w), (pad(x), pad(w))):
        leaves = [t.detach().requires_grad_() for t in (xx, ww, b)]
        h = ops.gated_linear(*leaves, activation="gelu")
        out.append([h.detach(), *torch.autograd.grad(h, leaves, dh)])
    (h, dx, dw, db), (h2, dx2, dw2, db2) = out
    want = gated_bounds(x, w, b, dh, "gelu", dtype)
    for name, a, c in (("h", h, h2), ("dx", dx, dx2[:, :D]), ("dw", dw, dw2[:, :D]), ("db", db, db2)):
        close(name, a, *want[name], dtype)
        close(name, c, *want[name], dtype)
    assert not dw2[:, D:].any()


def test_layer_norm_more_rows_than_one_grid_dimension_holds():
    M, C = (1 << 29) + 37, 2   # 8 lanes a row: over 2^32 threads
    x = torch.zeros(M, C, device="cuda", dtype=BF16)
    x[-100:] = _randn(_gen(46), 100, C, dtype=BF16)
    x.requires_grad_()
    y = ops.layer_norm(x, eps=0.5)
    (dx,) = torch.autograd.grad(y, x, x.detach())
    t = x.detach()[-100:].clone().requires_grad_()
    z = ops.layer_norm(t, eps=0.5)
    (dt,) = torch.autograd.grad(z, t, t.detach())
    assert t.any() and torch.equal(y[-100:], z) and torch.equal(dx[-100:], dt)
    assert not y[:-100].any() and not dx[:-100].any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gated_linear_rows_far_apart(dtype):
    """Rows further apart than a tile can address are copied."""
    g = _gen(47)
    for M in (3, 40):
        x, w, b, dh = _gated_inputs(g, M, 24, 16, dtype)
        far = torch.zeros(M * 2_000_016, device="cuda", dtype=dtype).as_strided((M, 24), (2_000_016, 1))
        far.copy_(x)
        out = []
        for t in (x, far):
            leaf = t.detach().requires_grad_()
            h = ops.gated_linear(leaf, w, b)
            out.append((h.detach(), *torch.autograd.grad(h, leaf, dh)))
        assert all(torch.equal(p, q) for p, q in zip(*out))


def test_parameters_with_strides():
    """Strided leaves: their gradients, and the refusal to capture beside a living graph of theirs."""
    g = _gen(48)
    x, dy = _randn(g, 20, 32), _randn(g, 20, 32)
    w, b, gw, gb = (t[..., ::2].requires_grad_() for t in (_randn(g, 64), _randn(g, 64), _randn(g, 64, 64), _randn(g, 128)))
    calls = (lambda w, b: ops.layer_norm(x, w, b), (w, b)), (lambda w, b: ops.gated_linear(x, w, b), (gw, gb))
    for call, leaves in calls:
        assert all(t.is_leaf and not t.is_contiguous() for t in leaves)
        alive = call(*leaves)
        dense = [t.detach().contiguous().requires_grad_() for t in leaves]
        want = torch.autograd.grad(call(*dense), dense, dy)
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call(*leaves)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(alive, leaves, dy), want))


def test_refused_on_the_gpu():
    x, w = torch.zeros(3, 4, device="cuda"), torch.zeros(6, 4, device="cuda")
    for bad in (torch.float16, torch.float64):
        with pytest.raises(TypeError):
            ops.layer_norm(x.to(bad))
        with pytest.raises(TypeError):
            ops.layer_norm(x, torch.ones(4, device="cuda", dtype=bad))
        with pytest.raises(TypeError):
            ops.dropout(x.to(bad), 0.1, 1)
        with pytest.raises(TypeError):
            ops.gated_linear(x.to(bad), w.to(bad))
    with pytest.raises(TypeError):
        ops.gated_linear(x, w.bfloat16())
    with pytest.raises(TypeError), torch.autocast("cuda", dtype=torch.float16):
        ops.gated_linear(x, w)
    with pytest.raises(ValueError):
        ops.layer_norm(x, torch.ones(4))
    with pytest.raises(ValueError):
        ops.gated_linear(x, w, torch.zeros(6))
    with pytest.raises(ValueError):
        ops.dropout(x, 0.1, 1, torch.tensor([1]))
