"""CPU: references, known answers and refusals of layer norm, counter-based dropout and the gated linear layer."""
import numpy as np
import pytest
import torch

from gsc_amd import ops
from gsc_amd.ops.philox_dropout import _philox, threshold
from tests.feedforward_bounds import close, gated_bounds, layer_norm_bounds


def test_philox_known_answers():
    """The generator's published vectors (key, counter all zeros / all ones)."""
    assert [hex(v) for v in _philox(1, 0, 0)[0]] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


def test_dropout_mask_rates_and_threshold():
    assert threshold(0.0) == 0 and threshold(0.5) == 1 << 31 and threshold(1 - 2.0 ** -40) == 2 ** 32 - 1
    n = 1 << 18
    for p in (0.0, 0.1, 0.5, 0.9):
        kept = int(ops.dropout_mask((n,), p, 3, 4).sum())
        assert abs(kept - (1 - p) * n) <= 6 * (n * p * (1 - p)) ** 0.5   # six standard deviations
    assert torch.equal(ops.dropout_mask((4, 25), 0.3, 3).view(-1), ops.dropout_mask((100,), 0.3, 3))


def test_dropout_cpu():
    x = torch.randn(10, 33, requires_grad=True)
    res = torch.randn(10, 33, requires_grad=True)
    y = ops.dropout(x, 0.25, 7, 3, residual=res)
    keep = ops.dropout_mask(x.shape, 0.25, 7, 3)
    assert torch.equal(y.detach(), torch.where(keep, x.detach() * (1 / 0.75), torch.zeros(())) + res.detach())
    dy = torch.randn(10, 33)
    dx, dres = torch.autograd.grad(y, (x, res), dy)
    assert torch.equal(dx, torch.where(keep, dy * (1 / 0.75), torch.zeros(()))) and torch.equal(dres, dy)
    assert torch.equal(ops.dropout(x, 0.25, 7, torch.tensor([3]), residual=res), y)
    bad = torch.full((64,), float("nan"))
    assert torch.equal(ops.dropout(bad, 0.5, 1, 1).isnan(), ops.dropout_mask((64,), 0.5, 1, 1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm_and_gated_linear_cpu(dtype):
    g = torch.Generator().manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype)
    x, w, b, dy = mk(7, 30).requires_grad_(), torch.rand(30, generator=g).requires_grad_(), mk(30).requires_grad_(), mk(7, 30)
    y = ops.layer_norm(x, w, b)
    want = layer_norm_bounds(x, w, b, dy, 1e-5)
    close("y", y, *want["y"], dtype)
    close("dx", torch.autograd.grad(y, x, dy)[0], *want["dx"], dtype)
    w2, b2 = (mk(24, 30) * 0.2).requires_grad_(), mk(24)
    for act in ("silu", "gelu", "sigmoid"):
        close("h", ops.gated_linear(x, w2, b2, activation=act), *gated_bounds(x, w2, b2, None, act, dtype)["h"], dtype)


def test_gradients_of_the_references():
    """The references' gradients against differences, in 64 bits."""
    g = torch.Generator().manual_seed(2)
    mk = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
    assert torch.autograd.gradcheck(ops.layer_norm, (mk(4, 9), mk(9), mk(9)))
    for act in ("silu", "gelu", "sigmoid"):
        assert torch.autograd.gradcheck(lambda x, w, b: ops.gated_linear(x, w, b, act), (mk(3, 5), mk(8, 5), mk(8)))
    assert torch.autograd.gradcheck(lambda x, r: ops.dropout(x, 0.3, 5, 1, residual=r), (mk(6, 7), mk(6, 7)))


def test_counted_bounds_are_of_the_right_size():
    """The bounds the GPU tests use are not vacuous: for bf16 outputs the fp32 part is below half the last rounding (2^-8)."""
    g = torch.Generator().manual_seed(3)
    x, w, dh = torch.randn(64, 64, generator=g), torch.randn(128, 64, generator=g) / 8, torch.randn(64, 64, generator=g)
    for k, (v, t) in gated_bounds(x, w, None, dh, "silu", torch.float32).items():
        assert t.norm() <= 2.0 ** -9 * v.norm(), k
    for k, (v, t) in layer_norm_bounds(x, None, None, dh, 1e-5).items():
        assert t.norm() <= 2.0 ** -9 * v.norm(), k


@pytest.mark.parametrize("call", [
    lambda t: ops.layer_norm(torch.zeros(())), lambda t: ops.layer_norm(t.new_zeros(3, 0)),
    lambda t: ops.layer_norm(t, torch.zeros(5)), lambda t: ops.layer_norm(t, None, torch.zeros(4, 1)),
    lambda t: ops.layer_norm(t, eps=-1.0), lambda t: ops.layer_norm(t, eps=float("nan")),
    lambda t: ops.dropout(t, 1.0, 1), lambda t: ops.dropout(t, -0.1, 1), lambda t: ops.dropout(t, float("nan"), 1),
    lambda t: ops.dropout(t, 0.1, -1), lambda t: ops.dropout(t, 0.1, 1 << 64), lambda t: ops.dropout(t, 0.1, 1, -1),
    lambda t: ops.dropout(t, 0.1, 1, 1 << 63), lambda t: ops.dropout(t, 0.1, 1, torch.tensor([-3])),
    lambda t: ops.dropout(t, 0.1, 1, residual=t[:1]), lambda t: ops.dropout(t, 0.1, 1, residual=t.double()),
    lambda t: ops.gated_linear(t, torch.zeros(6, 4), activation="relu"), lambda t: ops.gated_linear(t, torch.zeros(5, 4)),
    lambda t: ops.gated_linear(t, torch.zeros(6, 3)), lambda t: ops.gated_linear(t, torch.zeros(0, 4)),
    lambda t: ops.gated_linear(t, torch.zeros(6, 4), torch.zeros(3)), lambda t: ops.gated_linear(torch.zeros(()), torch.zeros(6, 4)),
    lambda t: ops.gated_linear(t, torch.zeros(6, 4), w16=torch.zeros(6, 4)),
    lambda t: ops.gated_linear(t, torch.zeros(6, 4), w16=torch.zeros(4, 4, dtype=torch.bfloat16))])
def test_refused_values(call):
    with pytest.raises(ValueError):
        call(torch.zeros(3, 4))


@pytest.mark.parametrize("call", [lambda t: ops.dropout(t, 0.1, 1, torch.tensor([1.0])),
                                  lambda t: ops.dropout(t, 0.1, 1, torch.tensor([1, 2]))])
def test_refused_types(call):
    with pytest.raises(TypeError):
        call(torch.zeros(3, 4))


def test_native_refusals():
    """What the kernels cannot address is refused on the host, before any launch."""
    nat = pytest.importorskip("gsc_amd.native").load()
    assert nat.gated_workspace(True, 100, 64, 256, True, True, True) >= 100 * 512 * 2
    for sizes in ((0, 8, 8), (8, 0, 8), (8, 8, 0), (8, 1_000_001, 8), (8, 8, 1_000_001), (1 << 31, 8, 8)):
        with pytest.raises(RuntimeError, match="gated_linear"):
            nat.gated_workspace(True, *sizes, True, True, True)
    call = lambda x, ldx: nat.gated_forward(x, ldx, 256, 8, True, 0, False, 256, 0, 4, 8, 4, 0, 0)
    for x, ldx in ((264, 8), (256, 12), (256, 2_000_008)):   # unaligned rows, rows too long for a descriptor
        with pytest.raises(RuntimeError, match="16-byte aligned rows"):
            call(x, ldx)
    with pytest.raises(RuntimeError, match="activation"):
        nat.gated_forward(256, 8, 256, 8, True, 0, False, 256, 0, 4, 8, 4, 3, 0)
    with pytest.raises(RuntimeError, match="layer_norm"):
        nat.layer_norm_forward(256, 8, True, 0, False, 0, False, 256, 0, 0, 0, 8, 1e-5, 0)
    for p in (1.0, -0.5, float("nan")):
        with pytest.raises(RuntimeError, match="dropout"):
            nat.dropout(256, 0, 256, True, 8, 1, 1, 0, 0, p, 0)


def test_native_refusals_of_layer_norm_sizes():
    nat = pytest.importorskip("gsc_amd.native").load()
    for M, C in ((0, 8), (8, 0), (1 << 31, 8), (8, (1 << 24) + 1)):
        with pytest.raises(RuntimeError, match="layer_norm"):
            nat.layer_norm_forward(256, 8, True, 0, False, 0, False, 256, 0, 0, M, C, 1e-5, 0)
        with pytest.raises(RuntimeError, match="layer_norm"):
            nat.LayerNormBackward(True, False, 0, M, C, False, False)
    assert nat.LayerNormBackward(True, False, 0, 1 << 20, 1 << 24, False, False).space <= 1 << 28   # 1 GB


def test_forward_workspace_of_gated_linear():
    """K is split, through a workspace, only where the tiles are few and K is long."""
    space = pytest.importorskip("gsc_amd.native").load().gated_forward_space
    assert space(True, 100, 4096, 256) > 0 and space(False, 100, 4096, 256) > 0
    for sizes in ((1, 4096, 256), (32, 4096, 256), (100, 128, 256), (200, 4096, 8192), (25600, 4096, 1024)):
        assert space(True, *sizes) == 0
    assert space(False, 25600, 4096, 1024) == 0
    with pytest.raises(RuntimeError, match="gated_linear"):
        space(True, 0, 8, 8)
