"""CPU: the cross-attention, sandwich-norm and Muon entries refuse what they cannot do before any HIP call, with a message; the formulas' plain
statements used by the GPU tests agree with differences."""
import ctypes

import pytest
import torch

from cross_reference import attention, sandwich

P = ctypes.c_void_p(4096)          # a device pointer that no refused call may touch


def _lib():
    from snag_amd import _lib
    return _lib.load(), _lib


def _fwd(dtype=1, B=2, Lq=3, Lk=5, H=4, Hkv=2, d=64, q=P, k=P, v=P, strides=True, lens=None, lens_bytes=4, mask=None, mask_ld=0, scale=0.125, out=P, lse=P, work=None, floats=0):
    lib, L = _lib()
    s = (ctypes.c_int64 * 9)(*([64] * 9))
    rc = lib.snag_cross_fwd(q, k, v, dtype, B, Lq, Lk, H, Hkv, d, ctypes.addressof(s) if strides else None, lens, lens_bytes, mask, mask_ld, scale, out, None, lse, work, floats, None)
    return rc, L.last_error()


@pytest.mark.parametrize("change, code, word", [
    (dict(dtype=3), -1, "dtype"), (dict(B=-1), -1, "size"), (dict(H=3), -1, "multiple"), (dict(Hkv=0), -1, "size"), (dict(d=0), -2, "head dimension"),
    (dict(d=129), -2, "head dimension"), (dict(q=None), -1, "null q"), (dict(k=None), -1, "null k"), (dict(v=None), -1, "null k"), (dict(strides=False), -1, "strides"),
    (dict(lens=P, lens_bytes=2), -1, "lens_bytes"), (dict(scale=0.0), -1, "scale"), (dict(scale=float("nan")), -1, "scale"), (dict(scale=float("inf")), -1, "scale"),
    (dict(scale=-1.0), -1, "scale"), (dict(out=None), -1, "null out"), (dict(lse=None), -1, "null out"), (dict(mask=P, mask_ld=-1), -1, "mask"),
    (dict(Lq=1 << 29, H=8, Hkv=2), -2, "2^30"), (dict(Lq=1, Lk=100000, B=1), -1, "workspace"),
    (dict(B=1 << 26, Lq=1, Lk=1), -2, "threads"), (dict(B=1 << 25, Lq=10, Lk=1), -2, "threads"), (dict(B=1 << 23, Lq=40, Lk=1), -2, "threads"),
])
def test_cross_attention_refusals(change, code, word):
    rc, text = _fwd(**change)
    assert rc == code and word in text, (rc, text)


def test_cross_attention_backward_refusals():
    lib, L = _lib()
    s = (ctypes.c_int64 * 9)(*([64] * 9))

    def bwd(out=P, lse=P, do=P, dq=P, dk=P, dv=P, work=None, floats=0):
        return lib.snag_cross_bwd(P, P, P, 1, 2, 3, 5, 4, 2, 64, ctypes.addressof(s), None, 4, None, 0, 0.1, out, None, lse, do, dq, dk, dv, work, floats, None), L.last_error()

    for change in ("out", "lse", "do", "dq", "dk", "dv"):
        rc, text = bwd(**{change: None})
        assert rc == -1 and "null" in text, (change, rc, text)
    rc, text = bwd()
    assert rc == -1 and "workspace" in text
    assert lib.snag_cross_work_floats(1, 2, 3, 5, 4, 2, 64, 1) >= 2 * 3 * 4
    assert lib.snag_cross_work_floats(1, 2, 3, 5, 4, 2, 200, 1) == 0          # refused by the call itself


def _sandwich(x=P, xt=1, y=P, yt=1, rows=6, dim=64, wt=1, gate=P, gt=1, rpg=3, kind=0, h=P, z=P, stats=None):
    lib, L = _lib()
    return lib.snag_sandwich_fwd(x, xt, y, yt, rows, dim, P, None, P, None, wt, gate, gt, rpg, 1.0, kind, 1e-6, h, z, stats, None), L.last_error()


@pytest.mark.parametrize("change, code, word", [
    (dict(yt=7), -1, "dtype"), (dict(xt=2), -2, "residual"), (dict(wt=2), -2, "weights"), (dict(gt=2), -2, "gate"), (dict(rows=-1), -1, "rows"), (dict(dim=0), -1, "rows"),
    (dict(dim=8193), -2, "width"), (dict(kind=2), -1, "kind"), (dict(rpg=4), -1, "multiple"), (dict(rpg=0), -1, "multiple"), (dict(x=None), -1, "null"), (dict(y=None), -1, "null"),
    (dict(h=None), -1, "null"), (dict(z=None), -1, "null"), (dict(stats=ctypes.c_void_p(4100)), -1, "aligned"),
])
def test_sandwich_norm_refusals(change, code, word):
    rc, text = _sandwich(**change)
    assert rc == code and word in text, (rc, text)


def test_sandwich_norm_backward_refusals():
    lib, L = _lib()

    def bwd(stats=P, dx=P, dy=P, gate=P, dgate=P, work=P, floats=1 << 20):
        return lib.snag_sandwich_bwd(P, 1, P, 1, 6, 64, P, None, P, 1, gate, 1, 3, 1.0, 0, stats, P, P, dx, dy, P, None, P, None, dgate, work, floats, None), L.last_error()

    for change, word in ((dict(stats=None), "null"), (dict(dx=None), "null"), (dict(dy=None), "null"), (dict(gate=None), "without"), (dict(work=None), "workspace"),
                         (dict(floats=10), "workspace"), (dict(stats=ctypes.c_void_p(4104)), "aligned")):
        rc, text = bwd(**change)
        assert rc == -1 and word in text, (change, rc, text)


def test_muon_refusals():
    lib, L = _lib()
    one = (ctypes.c_void_p * 1)(4096)
    none = (ctypes.c_void_p * 1)(None)
    shape = lambda n: (ctypes.c_int32 * 1)(n)
    A = ctypes.addressof

    def orth(g=one, out=one, r=8, c=8, count=1, dtype=1, steps=5, eps=1e-7, work=ctypes.c_void_p(4096), nbytes=1 << 30):
        rows, cols = shape(r), shape(c)
        return lib.snag_orthogonalize(A(g), A(out), A(rows), A(cols), count, dtype, steps, eps, work, nbytes, None), L.last_error()

    for change, code, word in ((dict(dtype=5), -1, "dtype"), (dict(r=0), -1, "0 x 8"), (dict(c=16385), -2, "longer"), (dict(count=-1), -1, "matrices"), (dict(steps=0), -1, "steps"),
                               (dict(steps=101), -1, "steps"), (dict(eps=-1.0), -1, "eps"), (dict(g=none), -1, "null matrix"), (dict(out=none), -1, "null matrix"),
                               (dict(work=None), -1, "workspace"), (dict(work=ctypes.c_void_p(4100)), -1, "workspace"), (dict(nbytes=1000), -1, "workspace")):
        rc, text = orth(**change)
        assert rc == code and word in text, (change, rc, text)
    assert orth(count=0)[0] == 0
    r, c = shape(8), shape(8)
    for mu in (-0.1, 1.0, float("nan")):
        rc = lib.snag_muon_step(A(one), A(one), A(one), A(r), A(c), 1, 1, 0.1, mu, 1, 0.0, 0, 5, 1e-7, 4096, 1 << 30, None)
        assert rc == -1 and "momentum" in L.last_error()
    assert lib.snag_muon_step(A(one), A(one), None, A(r), A(c), 1, 1, 0.1, 0.9, 1, 0.0, 0, 5, 1e-7, 4096, 1 << 30, None) == -1


def test_ops_refuse_cpu_tensors():
    from snag_amd import _lib, ops
    t, m = torch.zeros(2, 3, 4, 8), torch.zeros(4, 4)
    with pytest.raises(_lib.SnagHipError):
        ops.cross_attention_fwd(t, t, t)
    with pytest.raises(_lib.SnagHipError):
        ops.sandwich_norm_fwd(t, t)
    with pytest.raises(_lib.SnagHipError):
        ops.orthogonalize([m])
    with pytest.raises(_lib.SnagHipError):
        ops.muon_step([m], [m], [m], 0.1)
    with pytest.raises(TypeError):
        ops.cross_attention_fwd(t.double(), t, t)
    assert ops.orthogonalize([]) == []


def test_constants_match_the_header():
    import os
    import re
    from snag_amd import ops
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "snag_hip.h")).read()
    value = lambda name: int(re.search(rf"#define\s+{name}\s+(\d+)", text).group(1))
    assert (value("SNAG_CROSS_MAX_HEAD_DIM"), value("SNAG_SANDWICH_MAX_DIM"), value("SNAG_MUON_MAX_SIDE")) == (ops.CROSS_MAX_HEAD_DIM, ops.SANDWICH_MAX_DIM, ops.MUON_MAX_SIDE)
    assert {value("SNAG_F32"): torch.float32, value("SNAG_BF16"): torch.bfloat16, value("SNAG_F16"): torch.float16} == {v: k for k, v in ops.DTYPES.items()}
    assert {"rms": value("SNAG_NORM_RMS"), "layer": value("SNAG_NORM_LAYER")} == ops.NORMS


def test_muon_optimizer_takes_matrices_only_and_set_optim_cuts_the_groups():
    import types
    from snag_amd.optim import Muon, set_optim
    with pytest.raises(ValueError, match="not a matrix"):
        Muon([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(3, 3))], momentum=1.0)
    model = torch.nn.Module()
    model.entity_emb, model.img_fc = torch.nn.Embedding(10, 4), torch.nn.Linear(6, 4)
    model.weight_raw = torch.nn.Parameter(torch.ones(6))
    opt = types.SimpleNamespace(model_name="SNAG", lr=1e-3, weight_decay=0.1, adam_epsilon=1e-8, optim="muon", scheduler="fixed", warmup_steps=0, total_steps=10,
                                accumulation_steps=1, muon_lr=0.02)
    o, _ = set_optim(opt, [model])
    where = {p: g for g in o.param_groups for p in g["params"]}
    assert len(where) == 4
    assert where[model.img_fc.weight]["muon"] and where[model.img_fc.weight]["lr"] == 0.02 and where[model.img_fc.weight]["weight_decay"] == 0.1
    for p, decay in ((model.entity_emb.weight, 0.1), (model.img_fc.bias, 0.0), (model.weight_raw, 0.0)):
        assert not where[p]["muon"] and where[p]["lr"] == 1e-3 and where[p]["weight_decay"] == decay


def test_plain_gradients_agree_with_differences():
    """The 64-bit statements the GPU tests compare against: gradient formulas against central differences."""
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    B, Lq, Lk, H, Hkv, d = 2, 3, 5, 4, 2, 3
    q, k, v, do = rnd(B, Lq, H, d), rnd(B, Lk, Hkv, d), rnd(B, Lk, Hkv, d), rnd(B, Lq, H, d)
    lens, mask = torch.tensor([5, 0]), torch.rand(B, Lk, generator=g) < 0.7
    ref = attention(q, k, v, lens, mask, 0.6, do)
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        for _ in range(6):
            e = torch.zeros_like(t).view(-1)
            e[torch.randint(0, t.numel(), (1,), generator=g)] = 1e-5
            e = e.view_as(t)
            args = {n: (x + s * e if x is t else x) for s in (1,) for n, x in (("q", q), ("k", k), ("v", v))}
            less = {n: (x - e if x is t else x) for n, x in (("q", q), ("k", k), ("v", v))}
            diff = ((attention(**args, lens=lens, mask=mask, scale=0.6)["o"] - attention(**less, lens=lens, mask=mask, scale=0.6)["o"]) * do).sum() / 2e-5
            assert abs(float(diff - (ref[name] * e).sum() / 1e-5)) < 1e-8, name
    p = dict(x=rnd(6, 5), y=rnd(6, 5), post_weight=rnd(5), pre_weight=rnd(5), post_bias=rnd(5), pre_bias=rnd(5), gate=rnd(2, 5))
    dh, dz = rnd(6, 5), rnd(6, 5)
    for kind in ("rms", "layer"):
        ref = sandwich(**p, res_scale=0.7, kind=kind, eps=1e-6, d_h=dh, d_z=dz)
        for name, t in p.items():
            e = torch.zeros_like(t).view(-1)
            e[torch.randint(0, t.numel(), (1,), generator=g)] = 1e-5
            e = e.view_as(t)
            up, dn = (sandwich(**{**p, name: t + s * e}, res_scale=0.7, kind=kind, eps=1e-6) for s in (1, -1))
            diff = (((up["h"] - dn["h"]) * dh).sum() + ((up["z"] - dn["z"]) * dz).sum()) / 2e-5
            assert abs(float(diff - (ref["d_" + name] * e).sum() / 1e-5)) < 1e-7, (kind, name)


def test_muon_optimizer_keeps_the_momentum_of_16_bit_matrices_in_fp32():
    from snag_amd.optim import Muon, _is_matrix
    w = [torch.nn.Parameter(torch.zeros(4, 6, dtype=t)) for t in (torch.bfloat16, torch.float16, torch.float32)]
    opt, again = Muon(w), Muon(w)
    for p in w:
        opt.state[p]["momentum_buffer"] = torch.rand(4, 6)
    again.load_state_dict(opt.state_dict())
    for p in w:
        m = again.state[p]["momentum_buffer"]
        assert m.dtype == torch.float32 and torch.equal(m, opt.state[p]["momentum_buffer"])
    wide = torch.empty(2, 16385, device="meta")
    assert not _is_matrix("fc.weight", wide) and _is_matrix("fc.weight", wide[:, :16384])


def test_muon_lists_that_share_memory():
    from snag_amd import ops
    a, b = torch.zeros(10, 4), torch.zeros(10, 4)
    ops._disjoint([a[:5], a[5:]], [b, b])
    ops._disjoint([], [a, a[2:]])
    for written, read in (([a, a], []), ([a[:5], a[4:]], []), ([a], [a]), ([a[3:5]], [a]), ([a, b], [b[9:]])):
        with pytest.raises(ValueError, match="twice"):
            ops._disjoint(written, read)
