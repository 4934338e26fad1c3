"""GPU: cross attention, the sandwich norm and the orthogonalisation at the calls where precision, infinities or a derivative can get lost."""
import math

import pytest
import torch

from cross_reference import attention, attention_bounds, half_step, orthogonalized, orthogonalized_in_fp16, tiny_step

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E32 = 2.0 ** -24


def make(B, Lq, Lk, H, Hkv, d, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    return r(B, Lq, H, d), r(B, Lk, Hkv, d), r(B, Lk, Hkv, d), r(B, Lq, H, d)


def _row_tolerances(q, k, v, do, scale, r):
    """Norms that the errors of one gradient row (d elements) stay below, in fp16.  Each of the second products' operands (p, d scores) is rounded once, by
    at most half a step u of its value, independently of the others: squares add up, u sqrt(sum ds^2 k^2) -- doubled, for the spread of a norm over d
    elements.  fp32 sums of d terms of either sign: sqrt(d) 2^-24 of the terms' magnitudes, doubled, taken at their worst over keys or rows.  The result is
    rounded once: u, and half a subnormal step.  None of it grows when d_out gets small."""
    u, f = half_step(q.dtype), torch.float64
    B, Lq, H, d = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    G, e = H // Hkv, 2 * math.sqrt(d) * E32
    heads = lambda t: t.to(f).abs().repeat_interleave(H // t.shape[2], dim=2).permute(0, 2, 1, 3).contiguous()
    share = lambda t: t.view(B, Hkv, G, Lk, d).sum(2).permute(0, 2, 1, 3)
    qa, ka, va, da = (heads(t) for t in (q, k, v, do))
    p, ds = r["p"], r["ds"].abs()
    dpa = da @ va.transpose(2, 3).contiguous() + (da * r["o"].permute(0, 2, 1, 3).abs()).sum(-1, keepdim=True)
    norm = lambda t: t.square().sum(-1).sqrt()
    pt, dt, pd = (t.transpose(2, 3).contiguous() for t in (p, ds, p * dpa))
    es = e * (qa @ ka.transpose(2, 3).contiguous() * scale).amax() + 32 * E32
    last = tiny_step(q.dtype) * math.sqrt(d)
    return {"dq": (2 * u * scale * norm(((ds * ds) @ (ka * ka)).sqrt()) + (e + es) * scale * norm((p * dpa) @ ka)).permute(0, 2, 1) + u * norm(r["dq"]) + last,
            "dk": 2 * u * scale * norm(share((dt * dt) @ (qa * qa)).sqrt()) + (e + es) * scale * norm(share(pd @ qa)) + u * norm(r["dk"]) + last,
            "dv": 2 * u * norm(share((pt * pt) @ (da * da)).sqrt()) + (e + es) * norm(share(pt @ da)) + u * norm(r["dv"]) + last}


@pytest.mark.parametrize("size", [(2, 40, 2100, 2, 1, 64), (1, 20, 2100, 1, 1, 64), (1, 200, 2100, 2, 2, 128), (2, 5, 4096, 1, 1, 75), (1, 700, 30, 1, 1, 64), (3, 70, 500, 4, 2, 32)])
@pytest.mark.parametrize("magnitude", [1e-5, 1e-4, 1e-3, 1.0, 1e3])
def test_fp16_gradients_of_any_magnitude(size, magnitude):
    """d scores are about p |d_out| sqrt(d): over a few thousand keys they lie below fp16's smallest step for ordinary gradients."""
    from snag_amd import ops
    q, k, v, do = make(*size, torch.float16, seed=21)
    do = (do.float() * magnitude).half()
    q, scale = q * 0.25, 0.5
    if magnitude > 1:
        q, scale = q * 50, 0.01                          # d scores above 65504 whose gradients are not
    out, lse, lo = ops.cross_attention_fwd(q, k, v, scale=scale, want_residual=True)
    got = ops.cross_attention_bwd(q, k, v, out, lse, do, scale=scale, out_residual=lo)
    r = attention(q, k, v, scale=scale, d_out=do)
    tol = _row_tolerances(q, k, v, do, scale, r)
    for name, t in zip(("dq", "dk", "dv"), got):
        off = (t.double() - r[name]).square().sum(-1).sqrt()
        assert bool((off <= tol[name]).all()), (name, float((off / tol[name]).max()), float(off.norm() / r[name].norm()))


def test_fp16_gradients_of_large_scores():
    """Values and gradients whose d scores pass 65504 although no gradient does."""
    from snag_amd import ops
    q, k, v, do = make(2, 40, 6, 2, 1, 64, torch.float16, seed=30)
    v, do, scale = v * 30, do * 1000, 1e-3
    out, lse, lo = ops.cross_attention_fwd(q, k, v, scale=scale, want_residual=True)
    got = ops.cross_attention_bwd(q, k, v, out, lse, do, scale=scale, out_residual=lo)
    r = attention(q, k, v, scale=scale, d_out=do)
    assert float(r["ds"].abs().max()) > 65504 and all(float(r[n].abs().max()) < 65504 for n in ("dq", "dk", "dv"))
    tol = _row_tolerances(q, k, v, do, scale, r)
    for name, t in zip(("dq", "dk", "dv"), got):
        off = (t.double() - r[name]).square().sum(-1).sqrt()
        assert bool((off <= tol[name]).all()), (name, float((off / tol[name]).max()))


def test_fp16_probabilities_of_many_keys():
    """Probabilities of 300000 keys lie below fp16's smallest normal number, d v -- under a gradient scaled up as in 16-bit training -- does not."""
    from snag_amd import ops
    q, k, v, do = make(1, 6, 300000, 1, 1, 64, torch.float16, seed=22)
    q, do = q * 0.1, do * 200
    out, lse, lo = ops.cross_attention_fwd(q, k, v, want_residual=True)
    _, _, dv = ops.cross_attention_bwd(q, k, v, out, lse, do, out_residual=lo)
    r = attention(q, k, v, d_out=do)
    tol = _row_tolerances(q, k, v, do, 0.125, r)["dv"]
    off = (dv.double() - r["dv"]).square().sum(-1).sqrt()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(2, 40, 70, 2, 1, 64), (2, 130, 70, 2, 2, 128), (2, 50, 100, 1, 1, 32), (2, 3, 70, 2, 2, 64), (2, 20, 45, 1, 1, 64), (2, 40, 70, 2, 1, 75)])
def test_infinity_at_the_last_key_and_row(size, dtype):
    """What pads a tile must not be a copy of a key or row that holds an infinity: 0 x inf is NaN where the sum is infinite."""
    from snag_amd import ops
    q, k, v, do = make(*size, dtype, seed=23)
    B, Lk = size[0], size[2]
    lens = torch.tensor([Lk, Lk - 7], device=DEV, dtype=torch.int32)
    for ln in (None, lens):
        ends = [Lk - 1, Lk - 1 if ln is None else Lk - 8]
        clean, lse, lo = ops.cross_attention_fwd(q, k, v, ln, want_residual=True)
        bad = v.clone()
        for b in range(B):
            bad[b, ends[b], :, 5] = float("inf")
        out, _ = ops.cross_attention_fwd(q, k, bad, ln)
        assert bool((out[..., 5] == float("inf")).all())
        others = [c for c in range(size[5]) if c != 5]
        assert torch.equal(out[..., others], clean[..., others])
        # the last row of each problem, its element 5: d v[.., 5] is infinite at every seen key and nothing else of d v changes
        ref = ops.cross_attention_bwd(q, k, v, clean, lse, do, ln, out_residual=lo)[2]
        worse = do.clone()
        worse[:, -1, :, 5] = float("inf")
        dv = ops.cross_attention_bwd(q, k, v, clean, lse, worse, ln, out_residual=lo)[2]
        for b in range(B):
            assert bool((dv[b, :ends[b] + 1, :, 5] == float("inf")).all()) and bool((dv[b, ends[b] + 1:] == 0).all())
        assert torch.equal(dv[..., others], ref[..., others])


def test_forward_mode_derivatives_are_refused():
    """A tangent has no formula here: it must not be dropped (a missing tangent reads as zero)."""
    import torch.autograd.forward_ad as forward_ad
    from snag_amd._lib import SnagHipError
    from snag_amd.cross import cross_attention, sandwich_norm
    q, k, v, t = make(1, 3, 3, 2, 2, 32, torch.float32, seed=24)
    x, w = torch.randn(5, 64, device=DEV), torch.ones(64, device=DEV)
    plain, norm = cross_attention(q, k, v), sandwich_norm(x, x, w, w, gate=w)
    with forward_ad.dual_level():
        for i in range(3):
            args = [forward_ad.make_dual(a, t) if i == j else a for j, a in enumerate((q, k, v))]
            with pytest.raises(SnagHipError, match="forward"):
                cross_attention(*args)
        for names in (("x",), ("y",), ("post_weight",), ("pre_weight",), ("gate",)):
            args = dict(x=x, y=x, post_weight=w, pre_weight=w, gate=w)
            args.update({n: forward_ad.make_dual(args[n], torch.ones_like(args[n])) for n in names})
            with pytest.raises(SnagHipError, match="forward"):
                sandwich_norm(**args)
        assert torch.equal(cross_attention(q, k, v), plain)
        assert all(torch.equal(a, b) for a, b in zip(sandwich_norm(x, x, w, w, gate=w), norm))
        with pytest.raises(RuntimeError):
            cross_attention(forward_ad.make_dual(q.clone().requires_grad_(True), t), k, v)


@pytest.mark.parametrize("rows, dim", [(45000, 128), (100003, 96), (30000, 600)])
def test_parameter_gradients_of_many_rows(rows, dim):
    """d pre_bias = sum of d_z over the rows: nothing but the order of the sum.  Serial fp32 sums of n terms of either sign lose up to 2^-24 sqrt(n / 2)
    of the result, each rounding at its largest; the kernel's chain (a worker's run of at most 30 rows, 16 workers' partials, a tree of 16, a tree of
    16 runs): sqrt(15 + 8 + 4 + 4) 2^-24 at most."""
    from snag_amd import ops
    g = torch.Generator(device=DEV).manual_seed(25)
    x, y, dz = (torch.randn(rows, dim, generator=g, device=DEV) for _ in range(3))
    w = torch.ones(dim, device=DEV)
    _, _, stats = ops.sandwich_norm_fwd(x, y, pre_bias=w)
    got = ops.sandwich_norm_bwd(x, y, stats, None, dz, pre_bias=w)[5]
    ref = dz.double().sum(0)
    off = float((got.double() - ref).norm() / ref.norm())
    run = {128: 11, 96: 25, 600: 30}[dim]
    assert off <= E32 * math.sqrt(run / 2 + 8 + 4 + 4), (off, E32 * math.sqrt(run / 2 + 16))


def test_a_layer_with_frozen_norms_is_not_captured_over_a_live_graph():
    """Only the check runs: the forward inside the capture is refused before any backward is."""
    from snag_amd._lib import SnagHipError
    from snag_amd.cross import CrossModalLayer
    layer = CrossModalLayer(64, 4).to(DEV)
    for n, p in layer.named_parameters():
        p.requires_grad = "norm" not in n
    x = torch.randn(5, 3, 64, device=DEV)
    h, _ = layer(x, x)
    with pytest.raises(SnagHipError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            layer(x, x)
    h.sum().backward()
    assert all(bool(torch.isfinite(p.grad).all()) for p in layer.parameters() if p.grad is not None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [(1, 40, 3000, 2, 1, 64), (1, 2, 300, 2, 2, 64), (1, 2, 3000, 2, 1, 100), (4100, 1, 300, 1, 1, 32), (2, 40, 400, 2, 2, 75), (2, 200, 400, 1, 1, 128), (1, 3, 3000, 1, 1, 33)])
def test_the_residual_holds_what_rounding_dropped(size, dtype):
    """Values around 3: out's own rounding is what is off, and out + residual is much nearer.  (p's rounding, independent from key to key, reaches the
    output as u |v| sqrt(sum p^2), below a sixteenth of u |o| over these hundreds of keys; the residual's own is u^2.)  One wave, several waves and
    several ranges a problem, whole and odd widths."""
    from snag_amd import ops
    q, k, v, _ = make(*size, dtype, seed=26)
    q, v = q * 0.5, (v.float() * 0.2 + 3).to(dtype)
    out, _, lo = ops.cross_attention_fwd(q, k, v, want_residual=True)
    ref = attention(q, k, v)["o"]
    alone, both = float((out.double() - ref).norm()), float((out.double() + lo.double() - ref).norm())
    assert both <= alone / 4, (alone, both)
    assert bool((lo.double().abs() <= half_step(dtype) * 1.001 * out.double().abs()).all())
    assert bool((lo != 0).any(-1).float().mean() > 0.9)


def test_long_cache_gradients_pass_32_bits():
    """Element offsets behind 2^31 in both directions, keys and values apart: the last sequence's 100 seen keys at the end of 2.3 G elements."""
    from snag_amd import ops
    B, Lk, H, d = 72, 250000, 1, 128
    k, v = (torch.zeros(B, Lk, H, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(27)
    k[-1, -100:], v[-1, -100:] = (torch.randn(100, H, d, generator=g, device=DEV).bfloat16() for _ in range(2))
    lens = torch.full((B,), 3, device=DEV, dtype=torch.int32)
    lens[-1] = Lk
    mask = torch.zeros(B, Lk, dtype=torch.bool, device=DEV)
    mask[:, :3] = True
    mask[-1] = False
    mask[-1, -100:] = True
    for rows in (1, 40):
        q, do = (torch.randn(B, rows, H, d, generator=g, device=DEV).bfloat16() for _ in range(2))
        out, lse, lo = ops.cross_attention_fwd(q, k, v, lens, mask, want_residual=True)
        dq, dk, dv = ops.cross_attention_bwd(q, k, v, out, lse, do, lens, mask, out_residual=lo)
        small = (q[-1:], k[-1:, -100:], v[-1:, -100:])
        r = attention(*small, d_out=do[-1:])
        b = attention_bounds(*small, None, None, None, do[-1:], r)
        for name, t in (("o", out[-1:]), ("dq", dq[-1:]), ("dk", dk[-1:, -100:]), ("dv", dv[-1:, -100:])):
            assert bool(((t.double() - r[name]).abs() <= b[name]).all()), (rows, name)
        assert bool((dk[-1, :-100] == 0).all()) and bool((dv[-1, :-100] == 0).all())
        assert bool((dk[:-1, 3:] == 0).all()) and bool((out[:-1] == 0).all())
        del out, lse, lo, dq, dk, dv


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(16384, 300), (90, 16384)])
def test_the_longest_side(shape, dtype):
    from snag_amd.optim import orthogonalize
    g = torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(28), device=DEV).to(dtype)
    x = orthogonalized(g)
    cost = float((orthogonalized_in_fp16(g, 1 if dtype == torch.bfloat16 else 2).double() - x).norm() / x.norm())
    assert float((orthogonalize(g).double() - x).norm() / x.norm()) <= 2 * cost + 2e-6 + half_step(dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_step_keeps_its_types_bits(dtype):
    """A weight of zero, so that the update is all there is of the new one: fp32 and fp16 matrices carry 22 bits through the products, bf16 ones 11."""
    from snag_amd.optim import muon_step
    shapes = [(128, 700), (700, 128), (300, 200), (64, 129)]
    g = torch.Generator(device=DEV).manual_seed(29)
    gs = [(torch.randn(r, c, generator=g, device=DEV) * 1e-3).to(dtype) for r, c in shapes]
    ws, ms = [torch.zeros_like(t) for t in gs], [torch.randn(r, c, generator=g, device=DEV) * 1e-3 for r, c in shapes]
    m64 = [m.double() for m in ms]
    muon_step(ws, gs, ms, 1.0, 0.9)
    for (r, c), w, d, m in zip(shapes, ws, gs, m64):
        u = 0.1 * d.double() + 0.9 * (0.9 * m + 0.1 * d.double())
        x = orthogonalized(u)
        cost = float((orthogonalized_in_fp16(u, 1 if dtype == torch.bfloat16 else 2).double() - x).norm() / x.norm())
        off = float((w.double() + math.sqrt(max(1, r / c)) * x).norm() / (math.sqrt(max(1, r / c)) * x.norm()))
        assert off <= 2 * cost + 2e-6 + half_step(dtype), ((r, c), off, cost)


def test_a_layer_without_states_or_tokens():
    from snag_amd.cross import CrossModalLayer
    torch.manual_seed(0)
    layer = CrossModalLayer(64, 4, state_dim=48, kv_heads=2, intermediate_size=96).to(DEV)
    for N, M, L in ((5, 3, 0), (0, 3, 7), (5, 0, 7)):
        x, states = torch.randn(N, M, 64, device=DEV, requires_grad=True), torch.randn(N, L, 48, device=DEV, requires_grad=True)
        h, z = layer(x, states)
        assert h.shape == z.shape == (N, M, 64) and bool(torch.isfinite(h).all())
        (h.sum() + z.square().sum()).backward()
        assert x.grad.shape == x.shape and states.grad.shape == states.shape
        for n, p in layer.named_parameters():
            assert bool(torch.isfinite(p.grad).all()), n
            if n.split(".")[0] in ("key", "value") or N * M == 0:
                assert bool((p.grad == 0).all()), n
        layer.zero_grad(set_to_none=True)
