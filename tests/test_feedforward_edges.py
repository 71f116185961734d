"""CPU: what the feed-forward operators do on the host -- row views, refusals, builds."""
import pytest
import torch
from torch.autograd import forward_ad

from gsc_amd import ops
from gsc_amd.ops.launch import check_forward_mode, check_not_traced, rows_of


@pytest.mark.parametrize("view", [lambda t: t.unfold(0, 8, 1)[:5], lambda t: t.unfold(0, 8, 1)[:9], lambda t: t[:40].view(8, 5).t(),
                                  lambda t: t[:8].expand(5, 8), lambda t: t[:5, None].expand(5, 8),
                                  lambda t: t.unfold(0, 8, 2)[:6].view(2, 3, 8), lambda t: t[:40].view(5, 8)])
@pytest.mark.parametrize("dtype", [None, torch.float32, torch.bfloat16])
def test_rows_are_contiguous_behind_a_cast(view, dtype):
    """What a kernel reads through (pointer, row stride) are the elements of the view, overlapping windows included."""
    t = view(torch.arange(64.0))
    rows = rows_of(t, t.shape[-1], dtype)
    assert rows.dtype == (dtype or t.dtype) and rows.stride(1) == 1
    read = torch.as_strided(rows, rows.shape, (rows.stride(0), 1))
    assert torch.equal(read, t.to(rows.dtype).reshape(-1, t.shape[-1]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("C", [1, 2, 7, 15, 30, 41, 320, 1003, 16395])
def test_layer_norm_of_equal_values_is_the_bias(C, dtype):
    values = torch.tensor([7.0, 300.0, 30000.0, 0.1, -1 / 3, 1e8, -1e-3, 0.0], dtype=dtype)
    b = torch.randn(C, generator=torch.Generator().manual_seed(C), dtype=dtype)
    y = ops.layer_norm(values[:, None].repeat(1, C), torch.full((C,), 2.0, dtype=dtype), b)
    assert torch.equal(y, b.expand_as(y))


def test_tangents_and_traces_are_noticed():
    x = torch.randn(3)
    check_forward_mode("op", x, None)
    with forward_ad.dual_level():
        check_forward_mode("op", x, None)
        dual = forward_ad.make_dual(x, torch.ones(3))
        with pytest.raises(NotImplementedError, match="op: forward-mode"):
            check_forward_mode("op", None, dual)
        for y in (ops.layer_norm(dual), ops.dropout(dual, 0.0, 1)):   # the CPU's forms carry it
            assert forward_ad.unpack_dual(y).tangent is not None
    check_forward_mode("op", dual)
    check_not_traced("op")

    def traced(t):
        check_not_traced("op")
        return t + 1

    with pytest.raises(RuntimeError, match="op: cannot be traced"):
        torch.jit.trace(traced, x)
