"""GPU: the sandwich norm (both directions) against its 64-bit statement.

Bounds: e = 2^-24.  A sum over a row runs over at most 32 values per thread and a tree of 8, so its error is below 48 e of the terms'
magnitudes; the two directions chain at most five such stages (256 e), each scaled by how much larger a row's terms are than the row itself
(kappa: |res_scale x| + |gate post| against h, |y| + |mean| against y's deviation).  Parameter gradients add the worst case of a sum over all
rows.  Each output is rounded once: half a step."""
import pytest
import torch

from cross_reference import half_step, sandwich, tiny_step

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("x", "y", "post_weight", "pre_weight", "post_bias", "pre_bias", "gate")


def make(rows, dim, yt, xt=None, wt=None, gt=None, gates=None, bias=True, weights=True, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    xt, wt, gt = xt or yt, wt or yt, gt or yt
    p = dict(x=(2 * r(rows, dim)).to(xt), y=(r(rows, dim) + 0.2).to(yt))
    p["post_weight"] = (1 + 0.2 * r(dim)).to(wt) if weights else None
    p["pre_weight"] = (1 + 0.2 * r(dim)).to(wt) if weights else None
    p["post_bias"] = (0.2 * r(dim)).to(wt) if bias else None
    p["pre_bias"] = (0.2 * r(dim)).to(wt) if bias else None
    p["gate"] = None if gates is None else (0.5 + 0.5 * r(*((dim,) if gates == 0 else (gates, dim)))).to(gt)
    return p, r(rows, dim).to(xt), r(rows, dim).to(yt)


def bounds(p, ref, dh, dz, kind, res_scale, eps):
    e = 2.0 ** -24
    c = lambda t, none: torch.full((1,), none, dtype=torch.float64, device=DEV) if t is None else t.double()
    x, y, D = p["x"].double(), p["y"].double(), p["x"].shape[-1]
    g = c(p["gate"], 1.0)
    if p["gate"] is not None and p["gate"].dim() == 2:
        g = g.repeat_interleave(x.shape[0] // g.shape[0], 0)
    mean = lambda t: t.mean(-1, keepdim=True)
    rms = lambda t: mean(t * t).sqrt()
    center = mean(y) if kind == "layer" else 0 * mean(y)
    ry = 1 / (mean((y - center) ** 2) + eps).sqrt()
    ny = (y - center) * ry
    post = ny.abs() * c(p["post_weight"], 1.0).abs() + c(p["post_bias"], 0.0).abs()
    parts = abs(res_scale) * x.abs() + g.abs() * post
    h = ref["h"]
    hc = mean(h) if kind == "layer" else 0 * mean(h)
    rh = 1 / (mean((h - hc) ** 2) + eps).sqrt()
    nh = (h - hc) * rh
    k = (torch.maximum(rms(parts) * rh, rms(y.abs() + center.abs()) * ry).clamp_min(1.0)) ** 2 * 256 * e
    spread = lambda t: t + rms(t)                        # an error anywhere in a row reaches all of it through the row's statistics
    out = {"h": k * spread(parts), "z": k * (spread(nh.abs() + parts * rh) * c(p["pre_weight"], 1.0).abs() + c(p["pre_bias"], 0.0).abs())}
    if dh is not None or dz is not None:
        dz = torch.zeros_like(h) if dz is None else dz.double()
        dh = torch.zeros_like(h) if dh is None else dh.double()
        t = dz.abs() * c(p["pre_weight"], 1.0).abs()
        nha = nh.abs() + parts * rh
        d = dh.abs() + rh * spread(t + nha * mean(t * nha) + mean(t))
        dp = d * g.abs()
        nya = ny.abs() + (y.abs() + center.abs()) * ry
        t2 = dp * c(p["post_weight"], 1.0).abs()
        rows = x.shape[0]
        n = lambda terms: ((k + (rows + 32) * e) * terms).sum(0)
        out.update(d_x=abs(res_scale) * k * spread(d), d_y=k * ry * spread(t2 + nya * mean(t2 * nya) + mean(t2)), d_post_weight=n(dp * nya), d_post_bias=n(dp),
                   d_pre_weight=n(dz.abs() * nha), d_pre_bias=n(dz.abs()))
        if p["gate"] is not None:
            terms = (k + (rows + 32) * e) * d * post
            out["d_gate"] = terms.sum(0) if p["gate"].dim() == 1 else terms.view(p["gate"].shape[0], -1, D).sum(1)
    return out


def check(p, dh, dz, kind, res_scale=0.8, eps=1e-6, what=""):
    from snag_amd import ops
    par = {n: p[n] for n in NAMES[2:]}
    h, z, stats = ops.sandwich_norm_fwd(p["x"], p["y"], **par, res_scale=res_scale, kind=kind, eps=eps)
    got = dict(zip(["d_" + n for n in NAMES], ops.sandwich_norm_bwd(p["x"], p["y"], stats, dh, dz, **par, res_scale=res_scale, kind=kind)))
    got.update(h=h, z=z)
    ref = sandwich(**p, res_scale=res_scale, kind=kind, eps=eps, d_h=dh, d_z=dz)
    b = bounds(p, ref, dh, dz, kind, res_scale, eps)
    for n, t in got.items():
        if t is None:
            assert n[2:] in NAMES and p[n[2:]] is None, n
            continue
        off = (t.double().view(ref[n].shape) - ref[n]).abs()
        tol = b[n] + half_step(t.dtype) * ref[n].abs() + tiny_step(t.dtype)
        assert bool((off <= tol).all()), f"{what} {n}: excess {float((off - tol).nan_to_num(nan=9e9).max()):.3e}"
    return got


DIMS = [(1, 1), (5, 7), (3, 64), (40, 100), (9, 128), (70, 132), (33, 256), (12, 300), (6, 513), (20, 768), (7, 1000), (5, 1028), (4, 2048), (6, 2050), (3, 4096), (3, 5000), (2, 8192)]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", DIMS)
def test_against_the_statement(size, dtype, kind):
    check(*make(*size, dtype, gates=0), kind=kind, what=f"{size}")


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("types", [(torch.bfloat16, torch.float32, torch.float32, torch.bfloat16), (torch.float16, torch.float32, torch.float16, torch.float32),
                                   (torch.bfloat16, torch.bfloat16, torch.float32, torch.float32)])
@pytest.mark.parametrize("size", [(30, 128), (30, 300), (24, 2048)])
def test_mixed_types(size, types, kind):
    yt, xt, wt, gt = types
    check(*make(*size, yt, xt, wt, gt, gates=6), kind=kind, what=f"{size} {types}")


@pytest.mark.parametrize("rows, dim, gates", [(60, 128, 60), (60, 128, 20), (60, 300, 1), (9000, 64, 3), (9000, 64, 3000), (9000, 64, 9000), (6000, 100, 2), (4500, 1100, 4500),
                                              (4500, 1100, 5), (4500, 1100, 900), (45000, 128, 0), (5000, 1030, None), (3, 40, None)])
def test_gates_and_many_rows(rows, dim, gates):
    check(*make(rows, dim, torch.float32, gates=gates, bias=gates != 5), kind="layer", what=f"{rows} x {dim}, {gates} gates")
    check(*make(rows, dim, torch.bfloat16, gates=gates, weights=gates != 3, bias=False), kind="rms", what=f"{rows} x {dim}, {gates} gates")


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_without_variance_missing_gradients_and_alignment(kind):
    p, dh, dz = make(12, 130, torch.float32, gates=4, seed=3)
    p["y"][3] = 0.0
    p["y"][5] = 1.5                                     # constant: nothing but eps under a layer norm's root
    p["x"][7] = 0.0
    check(p, dh, dz, kind, eps=1e-3, what="flat rows")
    full = check(p, dh, dz, kind)
    assert all(bool(torch.isfinite(t).all()) for t in full.values())
    no_h = check(p, None, dz, kind, what="no d_h")
    no_z = check(p, dh, None, kind, what="no d_z")
    assert bool((no_z["d_pre_weight"] == 0).all()) and bool((no_z["d_pre_bias"] == 0).all()) and bool((no_h["d_pre_bias"] != 0).any())
    # dense tensors whose base is not 16-byte aligned
    for dtype in (torch.float32, torch.bfloat16):
        q, dh, dz = make(8, 128, dtype, gates=2)
        odd = lambda t: None if t is None else torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
        check({n: odd(t) for n, t in q.items()}, odd(dh), odd(dz), kind, what="odd base")


def test_differentiable_repeats_and_graph():
    from snag_amd._lib import SnagHipError
    from snag_amd.cross import sandwich_norm
    p, dh, dz = make(48, 256, torch.bfloat16, torch.float32, torch.float32, torch.bfloat16, gates=16)
    leaves = [p[n].requires_grad_(True) for n in NAMES]

    def all_of():
        h, z = sandwich_norm(p["x"].view(4, 12, 256), p["y"].view(4, 12, 256), *leaves[2:], res_scale=0.5, kind="layer")
        return [h.detach(), z.detach(), *torch.autograd.grad((h, z), leaves, (dh.view(h.shape), dz.view(z.shape)))]

    want = all_of()
    ref = sandwich(**p, res_scale=0.5, kind="layer", d_h=dh, d_z=dz)
    for n, t in zip(NAMES, want[2:]):
        assert t.dtype == p[n].dtype and t.shape == p[n].shape
        assert float((t.double() - ref["d_" + n]).norm() / ref["d_" + n].norm()) < (2.0 ** -8 if t.dtype == torch.bfloat16 else 1e-5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = all_of()
    for i in range(4):
        for t in got:
            t.zero_()
        graph.replay()
        junk = torch.randn(1 << 20, device=DEV)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), i
        assert all(torch.equal(a, b) for a, b in zip(want, all_of()))
    del junk
    alive = sandwich_norm(p["x"], p["y"], *leaves[2:])
    with pytest.raises(SnagHipError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            sandwich_norm(p["x"], p["y"], *leaves[2:])
    torch.autograd.grad(alive, leaves, (dh, dz))
    # one output only; no gradient wanted at all
    h, z = sandwich_norm(p["x"], p["y"], *leaves[2:])
    (only,) = torch.autograd.grad(z, leaves[1], dz)
    ref = sandwich(**p, kind="rms", d_z=dz)
    assert float((only.double() - ref["d_y"]).norm() / ref["d_y"].norm()) < 2.0 ** -8
    with torch.no_grad():
        h2, z2 = sandwich_norm(p["x"], p["y"], *leaves[2:])
    assert torch.equal(h, h2) and torch.equal(z, z2)


def test_empty_and_refusals():
    from snag_amd import ops
    from snag_amd.cross import sandwich_norm
    x = torch.zeros(0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    h, z = sandwich_norm(x, x, w, w, gate=w)
    assert h.shape == z.shape == (0, 64)
    gx, gw = torch.autograd.grad((h, z), (x, w), (torch.zeros_like(h), torch.zeros_like(z)))
    assert gx.shape == (0, 64) and bool((gw == 0).all())
    a, b = torch.zeros(6, 64, device=DEV), torch.zeros(6, 64, device=DEV).bfloat16()
    w16 = torch.ones(64, device=DEV).half()
    for args, kw, err in (((b, a), {}, TypeError), ((a, a[:5]), {}, ValueError), ((a, a), dict(kind="batch"), ValueError), ((a, a, w16), {}, TypeError), ((b, b, w16), {}, TypeError),
                          ((a, a), dict(gate=torch.ones(4, 64, device=DEV)), ValueError), ((a, a), dict(gate=torch.ones(1, 6, 64, device=DEV)), ValueError),
                          ((a, a, torch.ones(63, device=DEV)), {}, ValueError), ((a.t(), a.t()), {}, ValueError), ((torch.zeros(2, 8200, device=DEV),) * 2, {}, ValueError),
                          ((b, b, torch.ones(64, device=DEV), torch.ones(64, device=DEV).bfloat16()), {}, TypeError)):
        with pytest.raises(err):
            ops.sandwich_norm_fwd(*args, **kw)


def test_more_rows_than_threads_of_a_launch():
    """2^27 rows, 32 threads each: the forward takes several launches.  Rows are independent: any part alone gives the same bits."""
    from snag_amd import ops
    rows, dim, per = (1 << 27) + 8, 4, 8
    g = torch.Generator(device=DEV).manual_seed(14)
    x, y = (torch.empty(rows, dim, device=DEV, dtype=torch.bfloat16).normal_(generator=g) for _ in range(2))
    gate = torch.randn(rows // per, dim, generator=g, device=DEV)
    h, z, _ = ops.sandwich_norm_fwd(x, y, gate=gate, res_scale=0.5, want_stats=False)
    for a, b in ((0, 64), ((1 << 22) - 16, (1 << 22) + 16), (1 << 26, (1 << 26) + 4096), (rows - 4096, rows)):
        hp, zp, _ = ops.sandwich_norm_fwd(x[a:b], y[a:b], gate=gate[a // per:b // per], res_scale=0.5, want_stats=False)
        assert torch.equal(h[a:b], hp) and torch.equal(z[a:b], zp), (a, b)
