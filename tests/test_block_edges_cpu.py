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
