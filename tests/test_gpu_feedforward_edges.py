"""GPU: values at the edges of the feed-forward operators' ranges, against 64-bit results."""
import pytest
import torch

from gsc_amd import ops
from tests.feedforward_bounds import close, gated_bounds

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
