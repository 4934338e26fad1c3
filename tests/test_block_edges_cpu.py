"""CPU: refusals and bookkeeping of cross attention, the sandwich norm and Muon that need no kernel: forward-mode tangents, captures, launch limits."""
import ctypes

import pytest
import torch


def test_forward_mode_tangents_are_not_dropped(monkeypatch):
    """With the kernels' wrappers replaced: a dual tensor does not require grad, and a call past the autograd function would lose its tangent."""
    import torch.autograd.forward_ad as forward_ad
    from snag_amd import cross, ops
    from snag_amd._lib import SnagHipError
    monkeypatch.setattr(ops, "cross_attention_fwd", lambda q, *a, **k: (q.detach().clone(), q.new_zeros(1)))
    monkeypatch.setattr(ops, "sandwich_norm_fwd", lambda x, y, *a, **k: (x.detach().clone(), y.detach().clone(), None))
    t = torch.zeros(1, 2, 1, 4)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, torch.ones_like(t))
        for args in ((dual, t, t), (t, dual, t), (t, t, dual)):
            with pytest.raises(SnagHipError, match="forward"):
                cross.cross_attention(*args)
        for args in ((dual, t), (t, dual), (t, t, dual), (t, t, None, dual), (t, t, None, None, None, None, dual)):
            with pytest.raises(SnagHipError, match="forward"):
                cross.sandwich_norm(*args)
        assert torch.equal(cross.cross_attention(t, t, t), t)
    assert torch.equal(cross.cross_attention(t, t, t), t) and torch.equal(cross.sandwich_norm(t, t)[0], t)


@pytest.mark.parametrize("B, Lq, Lk, dtype, d", [(1 << 20, 5, 2048, 1, 64), (1 << 24, 9, 129, 0, 128), (1 << 22, 2048, 5, 2, 64), (1 << 26, 5, 1, 1, 32), (1 << 26, 0, 5, 1, 32)])
def test_a_backward_past_the_launch_limit_is_refused_before_anything_is_launched(B, Lq, Lk, dtype, d):
    """Too many waves on the keys' or on the rows' side, whichever the other one needs: nothing may be written first (without a device a launch
    answers with another error)."""
    from snag_amd import _lib
    lib, P = _lib.load(), ctypes.c_void_p(4096)
    strides = (ctypes.c_int64 * 9)(*([64] * 9))
    rc = lib.snag_cross_bwd(P, P, P, dtype, B, Lq, Lk, 1, 1, d, ctypes.addressof(strides), None, 4, None, 0, 0.1, P, None, P, P, P, P, P, P, 1 << 62, None)
    assert rc == -2 and "threads" in _lib.last_error(), (rc, _lib.last_error())


@pytest.mark.parametrize("r, c", [(2 ** 31 - 1, 2 ** 31 - 1), (16385, 8), (8, 2 ** 31 - 1), (0, 8), (8, -1)])
def test_no_workspace_is_computed_for_a_refused_matrix(r, c):
    """Sides past the limit are refused by the call; sizing their workspace would overflow 32-bit tile counts."""
    from snag_amd import _lib
    rows, cols = (ctypes.c_int32 * 2)(8, r), (ctypes.c_int32 * 2)(8, c)
    size = lambda n: _lib.load().snag_muon_work_bytes(ctypes.addressof(rows), ctypes.addressof(cols), n)
    assert size(2) == 0 and size(1) > 0


@pytest.fixture
def streams(monkeypatch):
    """The stream and whether it is capturing, as the test says."""
    from snag_amd import ops
    now = {"stream": 1, "capturing": False}
    monkeypatch.setattr(ops, "_raw_stream", lambda index: now["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    return now


def test_a_capture_over_leaves_of_a_live_eager_graph_is_refused_at_any_depth(streams):
    from snag_amd import cross
    from snag_amd._lib import SnagHipError
    w, other = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    alive = w * 2
    cross._note_stream(alive)
    streams.update(stream=2, capturing=True)
    for depth in range(4):
        t = w
        for _ in range(depth):
            t = t.view(3).clone()
        with pytest.raises(SnagHipError, match="eager graph"):
            cross._note_stream((t + other) * other if depth else t * other)
        cross._note_stream((other.view(3).clone() + 1) * other)
    del alive, t
    cross._note_stream(w.view(3).clone() * 2)                       # the eager graph is gone, and its nodes with it
    streams.update(stream=1, capturing=False)
    cross._note_stream(w * other)


def test_a_layer_notes_the_leaves_of_its_projections(streams, monkeypatch):
    """With its norms frozen the projections' weights are all that an eager graph and a captured one share."""
    from snag_amd import cross, ops, projection
    from snag_amd._lib import SnagHipError

    def gemm(a, b, bias=None, act=None, **_):
        r = a @ b.T if bias is None else a @ b.T + bias
        return r.relu() if act == "relu" else r

    monkeypatch.setattr(ops, "gemm", gemm)
    monkeypatch.setattr(cross, "cross_attention", lambda q, k, v, *_: q + k.mean() + v.mean())
    monkeypatch.setattr(cross, "sandwich_norm", lambda x, y, *_, **__: (x + y, x - y))
    for frozen in ([], ["query", "key", "value"], ["query", "key", "output", "feed_forward"], ["query", "key", "value", "output"]):
        layer = cross.CrossModalLayer(8, 2)
        for n, p in layer.named_parameters():
            p.requires_grad = n.split(".")[0] not in frozen and "norm" not in n
        x = torch.randn(2, 3, 8)
        streams.update(stream=1, capturing=False)
        alive = layer(x, x)
        streams.update(stream=2, capturing=True)
        with pytest.raises(SnagHipError, match="eager graph"):
            layer(x, x)
        del alive
        layer(x, x)


@pytest.mark.parametrize("side, padded, ranges", [(2600, 2688, 2 * 231), (4360, 4480, 4 * 118), (3400, 3584, 0), (3700, 3840, 0)])
def test_the_large_tile_is_taken_where_its_rounds_are_done_first(side, padded, ranges):
    """Seen from outside by the workspace (X, A and B: 16 bytes an element of the padded square; partial tiles of 64 KB): 2600 x 2600 are 121 tiles of 256,
    a whole round of the chip for less than half of it, or 441 of 128, one round of 512; 4360 x 4360 two rounds or three half as long; 3400 x 3400 and
    3700 x 3700 one or two half as long."""
    from snag_amd import _lib
    n = (ctypes.c_int32 * 1)(side)
    got = _lib.load().snag_muon_work_bytes(ctypes.addressof(n), ctypes.addressof(n), 1)
    assert 0 <= got - 16 * padded ** 2 - 65536 * ranges < 65536, got
