"""CPU: what the feed-forward operators do on the host -- row views, refusals, builds."""
import sys

import pytest
import torch
from torch.autograd import forward_ad

from gsc_amd import ops
from gsc_amd.ops import launch
from gsc_amd.ops.launch import check_forward_mode, check_leaves, check_not_traced, rows_of


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


def test_objects_of_another_command_are_compiled_again(tmp_path, monkeypatch):
    """An object is current when it is newer than its sources and its command line (flags, target, compiler) is the same."""
    from gsc_amd.native import build as b
    csrc, ran = tmp_path / "csrc", []
    csrc.mkdir()
    (csrc / "a.hip").write_text('#include "a.h"\n')
    (csrc / "a.h").write_text("\n")
    (tmp_path / "cc").write_text("#!/bin/sh\nwhile [ $# -gt 1 ]; do [ \"$1\" = -o ] && touch \"$2\"; shift; done\n")
    (tmp_path / "cc").chmod(0o755)
    for name, value in (("CSRC", str(csrc)), ("BUILD", str(tmp_path / "obj")), ("HIPCC", str(tmp_path / "cc")),
                        ("ext_path", lambda sanitize=False: str(tmp_path / "out.so"))):
        monkeypatch.setattr(b, name, value)
    run = b.subprocess.run
    monkeypatch.setattr(b.subprocess, "run", lambda cmd, **k: (ran.append("-c" in cmd), run(cmd, **k))[1])

    def made(**k):
        ran.clear()
        b.build(verbose=False, **k)
        return ran.count(True), ran.count(False)   # compiled, linked

    assert made() == (1, 1) and made() == (0, 0)
    flags = b._flags
    monkeypatch.setattr(b, "_flags", lambda src: flags(src) + ["-DX"])
    assert made()[0] == 1 and made() == (0, 0)
    monkeypatch.setattr(b, "ARCH", "gfx942")
    assert made() == (1, 1) and made() == (0, 0)
    later = (tmp_path / "out.so").stat().st_mtime + 10
    b.os.utime(csrc / "a.h", (later, later))
    assert made()[0] == 1
    b.os.utime(csrc / "a.h", (1, 1))
    assert made(force=True) == (1, 1) and made() == (0, 0)
    (tmp_path / "cc").write_text("#!/bin/sh\nexit 1\n")   # a failing compiler leaves nothing current
    with pytest.raises(RuntimeError, match="hipcc failed"):
        made(force=True)
    with pytest.raises(RuntimeError, match="hipcc failed"):
        made()


def test_the_entry_point_compiles_every_source(monkeypatch):
    import __graft_entry__
    from gsc_amd.native import build as b
    seen = []
    monkeypatch.setattr(b, "build", lambda **k: seen.append(k))
    pytest.importorskip("gsc_amd.native").load()
    __graft_entry__.build()
    assert seen == [{"verbose": True, "force": True}]


def test_workspaces_of_other_sizes_are_refused():
    """On the host, before any launch: the pointers are never read."""
    nat = pytest.importorskip("gsc_amd.native").load()
    M, D, F = 100, 4096, 256
    need, kept = nat.gated_forward_space(True, M, D, F), nat.gated_saved_elements(True, M, D, F)
    back = nat.gated_workspace(True, M, D, F, True, True, True)
    assert need > 0 and kept > 0

    def forward(saved, saved_size, work, work_size, sizes=(M, D, F)):
        nat.gated_forward_split(256, D, 256, D, True, 0, False, 256, saved, saved_size, work, work_size, *sizes, 0, 0)

    for work, work_size in ((0, 0), (0, need), (256, need - 1), (256, nat.gated_forward_space(True, M - 40, D, F) // 2)):
        with pytest.raises(RuntimeError, match="too little workspace for the forward pass"):
            forward(256, kept, work, work_size)
    with pytest.raises(RuntimeError, match="too little space for the kept products"):
        forward(256, kept - 1, 256, need)
    with pytest.raises(RuntimeError, match="not kept"):
        forward(256, 1 << 40, 256, 1 << 40, (M, 64, F))
    with pytest.raises(RuntimeError, match="keeps no products"):
        nat.gated_forward(256, D, 256, D, True, 0, False, 256, 256, M, D, F, 0, 0)

    def backward(saved, saved_size, work, work_size, act=0):
        nat.gated_backward(256, D, 256, D, True, 0, False, 256, F, saved, saved_size, 256, True, 256, True, 256, True, work,
                           work_size, M, D, F, act, 0)

    for work, work_size in ((0, back), (256, back - 1)):
        with pytest.raises(RuntimeError, match="too little workspace for the backward pass"):
            backward(256, kept, work, work_size)
    with pytest.raises(RuntimeError, match="too few kept products"):
        backward(256, kept - 1, 256, back)
    with pytest.raises(RuntimeError, match="kept products"):
        backward(0, 0, 256, back)
    with pytest.raises(RuntimeError, match="activation"):
        backward(256, kept, 256, back, act=3)


def test_leaves_held_by_graphs_of_another_stream(monkeypatch):
    """While capturing: a leaf that any operator's graph holds is refused unless that graph's stream is the captured one."""
    node, here, capturing = 5, 5, True
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    # the hook in the node asks for its stream, the check for the captured one
    monkeypatch.setattr(launch, "raw_stream", lambda dev: node if sys._getframe(1).f_code.co_name == "look" else here)
    w, x = torch.randn(3, requires_grad=True), torch.randn(3)
    check_leaves("op", x, None, w)               # no graph
    alive = w * 2
    check_leaves("op", x, None, w)               # a graph of this stream
    node = 6
    with pytest.raises(RuntimeError, match="op: a graph of the same leaf"):
        check_leaves("op", x, None, w)
    assert w.grad is None and torch.equal(torch.autograd.grad(alive, w, x, retain_graph=True)[0], 2 * x)   # left as it was
    check_leaves("op", alive)                    # not a leaf
    capturing = False
    check_leaves("op", w)
    capturing = True
    del alive
    check_leaves("op", w)
    called = []
    handle = w.register_hook(called.append)
    check_leaves("op", w)
    alive = w * 2
    with pytest.raises(RuntimeError, match="op: a graph"):   # its hooks are not called to find out
        check_leaves("op", w)
    assert not called
    handle.remove()


def test_few_tiles_are_split_only_where_the_partial_results_cost_less():
    """Writing and reading them counts: 300 x 2048 x 1024 takes 20 us in one piece, 23 in six."""
    nat = pytest.importorskip("gsc_amd.native").load()
    slab = lambda M, F: -(-M // 128) * 128 * -(-F // 64) * 128
    assert nat.gated_forward_space(True, 300, 2048, 1024) == 0
    assert nat.gated_forward_space(True, 512, 4096, 1024) == 4 * slab(512, 1024)
    assert nat.gated_forward_space(True, 100, 4096, 256) == 7 * slab(100, 256)
