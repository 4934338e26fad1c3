"""GPU: cross attention (both directions) against its 64-bit statement, at the sizes, layouts and masks where it can go wrong.  The bounds are
those of cross_reference.attention_bounds: every rounding counted at half a step, every fp32 sum at its worst case."""
import pytest
import torch

from cross_reference import attention, attention_bounds, half_step

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [  # B, Lq, Lk, H, Hkv, d
    (1, 1, 1, 1, 1, 1), (2, 1, 37, 4, 1, 64), (3, 2, 130, 4, 2, 128), (5, 3, 24, 2, 2, 64), (2, 1, 70, 3, 1, 40), (2, 4, 9, 1, 1, 33), (1, 1, 5000, 4, 2, 64),
    (1, 2, 3000, 2, 1, 100), (300, 3, 5, 2, 2, 32), (2, 7, 5, 3, 1, 32), (1, 33, 65, 2, 2, 64), (2, 129, 200, 4, 2, 128), (1, 40, 300, 2, 1, 75), (1, 5, 2000, 2, 1, 40),
    (1, 700, 3, 2, 2, 128), (2, 64, 64, 2, 1, 17), (1, 31, 33, 1, 1, 96), (3, 257, 129, 1, 1, 64), (1, 9, 1, 2, 1, 8), (1, 300, 1200, 2, 1, 64),
]


def make(B, Lq, Lk, H, Hkv, d, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    return r(B, Lq, H, d), r(B, Lk, Hkv, d), r(B, Lk, Hkv, d), r(B, Lq, H, d)


def check(q, k, v, do, lens=None, mask=None, scale=None, what=""):
    from snag_amd import ops
    out, lse, lo = ops.cross_attention_fwd(q, k, v, lens, mask, scale, want_residual=True)
    grads = ops.cross_attention_bwd(q, k, v, out, lse, do, lens, mask, scale, lo)
    r = attention(q, k, v, lens, mask, scale, do)
    b = attention_bounds(q, k, v, lens, mask, scale, do, r)
    for name, t in (("o", out), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        off = (t.double() - r[name]).abs()
        bad = ~(off <= b[name])
        assert not bool(bad.any()), f"{what} {name}: {int(bad.sum())} values outside, largest excess {float((off - b[name]).nan_to_num(nan=9e9).max()):.3e}"
    natural = lse.double() * 0.6931471805599453
    empty = r["lse"] == -float("inf")
    assert bool((lse[empty] == -float("inf")).all())
    assert bool(((natural - r["lse"]).abs() <= b["lse"] + 2.0 ** -24 * r["lse"].abs())[~empty].all()), f"{what} lse"
    return out, grads, r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_against_the_statement(size, dtype):
    check(*make(*size, dtype), what=str(size))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(3, 5, 300, 2, 2, 64), (2, 3, 1100, 2, 1, 100), (1, 7, 40, 1, 1, 128), (2, 2, 5000, 4, 1, 64), (300, 1, 9, 8, 1, 32), (1, 6, 1, 1, 1, 3), (40, 1, 333, 16, 2, 75),
                                  (2, 30, 4000, 1, 1, 128), (1, 60, 700, 2, 2, 40)])
def test_between_few_rows_and_a_tile(size, dtype):
    check(*make(*size, dtype, seed=16), what=str(size))
    q, k, v, do = make(*size, dtype, seed=17)
    B, Lk = size[0], size[2]
    lens = torch.tensor([(i * 7 + Lk) % (Lk + 1) for i in range(B)], device=DEV, dtype=torch.int64)
    g = torch.Generator(device=DEV).manual_seed(18)
    mask = torch.rand(B, Lk, generator=g, device=DEV) > 0.3
    unseen = ~mask | (torch.arange(Lk, device=DEV) >= lens[:, None])
    k[unseen], v[unseen] = float("nan"), float("inf")
    from snag_amd import ops
    out, lse, lo = ops.cross_attention_fwd(q, k, v, lens, mask, want_residual=True)
    got = ops.cross_attention_bwd(q, k, v, out, lse, do, lens, mask, out_residual=lo)
    k[unseen], v[unseen] = 0.0, 0.0
    ref_out, ref, _ = check(q, k, v, do, lens, mask, what=f"{size} masked")
    assert torch.equal(out, ref_out) and all(torch.equal(a, b) for a, b in zip(got, ref))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(6, 1, 70, 4, 2, 64), (6, 3, 24, 2, 2, 64), (6, 50, 70, 4, 2, 64), (6, 130, 140, 2, 2, 128), (6, 20, 1500, 2, 1, 64), (6, 2, 3000, 2, 1, 64)])
def test_lengths_and_masks_with_anything_behind_them(size, dtype):
    """Lengths 0, 1, whole and beyond; a mask that leaves a sequence nothing; NaN and infinities at every key that is not seen."""
    q, k, v, do = make(*size, dtype, seed=1)
    B, Lk = k.shape[:2]
    lens = torch.tensor([0, 1, Lk, Lk // 2, Lk + 9, -3], device=DEV)
    mask = torch.rand(B, Lk, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV) < 0.6
    mask[2] = False
    for ln, m in ((lens.int(), None), (lens, mask), (None, mask)):
        seen = torch.ones(B, Lk, dtype=torch.bool, device=DEV)
        if ln is not None:
            seen &= torch.arange(Lk, device=DEV)[None] < ln[:, None]
        if m is not None:
            seen &= m
        k2, v2 = k.clone(), v.clone()
        k2[~seen], v2[~seen] = float("nan"), float("inf")
        out, (dq, dk, dv), _ = check(q, k2, v2, do, ln, m, what=f"{size}")
        nothing = ~seen.any(1)
        assert bool((out[nothing] == 0).all()) and bool((dq[nothing] == 0).all())
        assert bool((dk[~seen] == 0).all()) and bool((dv[~seen] == 0).all())
        clean = check(q, torch.where(seen[..., None, None], k, 0), torch.where(seen[..., None, None], v, 0), do, ln, m)
        assert torch.equal(out, clean[0]) and all(torch.equal(a, b) for a, b in zip((dq, dk, dv), clean[1]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 40])
def test_strides_and_alignment(rows, dtype):
    """Heads in front, fused key/value projections, rows that are not 16-byte aligned, an expanded batch: the same bits as dense copies."""
    from snag_amd import ops
    B, Lk, H, d = 2, 50, 2, 64
    g = torch.Generator(device=DEV).manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    q = r(B, H, rows, d).transpose(1, 2)
    kv = r(B, Lk, 2, H, d)
    odd = r(B * Lk * H * d + 1)[1:].view(B, Lk, H, d)
    wide = r(B, Lk, H, d + 3)[..., :d]
    shared = r(1, Lk, H, d).expand(B, Lk, H, d)
    do = r(B, rows, H, d)
    mask = (torch.rand(B, 2 * Lk, generator=g, device=DEV) < 0.7)[:, 3:3 + Lk]
    for k, v in ((kv[:, :, 0], kv[:, :, 1]), (odd, kv[:, :, 1]), (wide, odd), (shared, wide)):
        out, (dq, dk, dv), _ = check(q, k, v, do, None, mask, what="strided")
        o2, l2, lo = ops.cross_attention_fwd(q.contiguous(), k.contiguous(), v.contiguous(), None, mask.contiguous(), want_residual=True)
        g2 = ops.cross_attention_bwd(q.contiguous(), k.contiguous(), v.contiguous(), o2, l2, do, None, mask.contiguous(), out_residual=lo)
        assert torch.equal(out, o2) and all(torch.equal(a, b) for a, b in zip((dq, dk, dv), g2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 40])
def test_large_scores_and_scale(rows, dtype):
    """Scores of several hundred (one key takes nearly all), and another scale."""
    q, k, v, do = make(2, rows, 90, 2, 1, 64, dtype, seed=3)
    check(q * 8, k * 4, v, do, what="large")
    check(q, k, v, do, scale=0.5, what="scale")
    check(q, k, v, do, scale=1e-4, what="flat")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("Lk", [1, 2, 3])
def test_few_keys_keep_their_gradient(Lk, rows, dtype):
    """Where p (do v^T - delta) cancels, the output's rounding must not reach delta: with the residual the gradients keep the type's precision.
    (Every rounding in the chain -- p or ds, q, k, the result -- is half a step; four of them, and the cancellation of fp32 sums.)"""
    from snag_amd import ops
    q, k, v, do = make(64, rows, Lk, 2, 2, 64, dtype, seed=8)
    out, lse, lo = ops.cross_attention_fwd(q, k, v, want_residual=True)
    got = ops.cross_attention_bwd(q, k, v, out, lse, do, out_residual=lo)
    r = attention(q, k, v, d_out=do)
    for name, t in zip(("dq", "dk", "dv"), got):
        off, size = float((t.double() - r[name]).norm()), float(r[name].norm())
        floor = 64 * 2.0 ** -24 * float(attention(q.abs(), k.abs(), v.abs(), d_out=do.abs())[name].norm() + do.double().norm() * v.double().norm() / 8)
        assert off <= 2 * half_step(dtype) * size + floor, (name, off, size, floor)


@pytest.mark.parametrize("dtype", TYPES)
def test_differentiable_and_empty(dtype):
    from snag_amd.cross import cross_attention
    q, k, v, do = (t.requires_grad_(i < 3) for i, t in enumerate(make(2, 5, 30, 4, 2, 32, dtype, seed=4)))
    lens = torch.tensor([30, 7], device=DEV, dtype=torch.int32)
    out, lse = cross_attention(q, k, v, lens, return_lse=True)
    r = attention(q.detach(), k.detach(), v.detach(), lens, None, None, do)
    b = attention_bounds(q.detach(), k.detach(), v.detach(), lens, None, None, do, r)
    for t, got in zip((q, k, v), torch.autograd.grad(out, (q, k, v), do)):
        name = "d" + {id(q): "q", id(k): "k", id(v): "v"}[id(t)]
        assert bool(((got.double() - r[name]).abs() <= b[name]).all())
    assert not lse.requires_grad and bool(((lse.double() - r["lse"]).abs() <= b["lse"] + 2.0 ** -22 * r["lse"].abs()).all())
    (only,) = torch.autograd.grad(cross_attention(q.detach(), k, v.detach(), lens), (k,), do)
    assert torch.equal(only, torch.autograd.grad(out := cross_attention(q, k, v, lens), (k,), do)[0])
    for B, Lq, Lk in ((0, 3, 4), (2, 0, 4), (2, 3, 0), (2, 50, 0)):
        q0, k0, v0 = (torch.randn(B, L, 2, 16, device=DEV, dtype=dtype, requires_grad=True) for L in (Lq, Lk, Lk))
        o = cross_attention(q0, k0, v0)
        assert o.shape == q0.shape and bool((o == 0).all())
        for t, got in zip((q0, k0, v0), torch.autograd.grad(o, (q0, k0, v0), torch.ones_like(o))):
            assert got.shape == t.shape and bool((got == 0).all())


def test_long_cache_offsets_pass_32_bits():
    """Element offsets behind 2^31: the last sequence of a key/value buffer of 2.3 G elements each."""
    from snag_amd import ops
    B, Lk, H, d = 72, 250000, 1, 128
    k = torch.zeros(B, Lk, H, d, device=DEV, dtype=torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(6)
    for rows in (1, 40):
        q = torch.randn(B, rows, H, d, generator=g, device=DEV).bfloat16()
        tail = torch.randn(2, 100, H, d, generator=g, device=DEV).bfloat16()
        k[-1, -100:] = tail[0]
        lens = torch.full((B,), 3, device=DEV, dtype=torch.int32)
        lens[-1] = Lk
        mask = torch.zeros(B, Lk, dtype=torch.bool, device=DEV)
        mask[:, :3] = True
        mask[-1] = False
        mask[-1, -100:] = True
        out, _ = ops.cross_attention_fwd(q, k, k, lens, mask)
        r = attention(q[-1:], k[-1:, -100:], k[-1:, -100:])
        b = attention_bounds(q[-1:], k[-1:, -100:], k[-1:, -100:], None, None, None, None, r)
        # the kernel adds up all 250000 keys, the bound's fp32 sums are of 100
        assert bool(((out[-1:].double() - r["o"]).abs() <= b["o"] + 2.0 ** -8 * r["o"].abs()).all())
        assert bool((out[:-1] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(3, 2, 70, 2, 2, 64), (3, 40, 70, 2, 1, 64), (3, 130, 200, 2, 2, 128)])
def test_gradients_of_rows_that_see_nothing_may_hold_anything(size, dtype):
    from snag_amd import ops
    q, k, v, do = make(*size, dtype, seed=12)
    lens = torch.tensor([size[2], 0, size[2] - 3], device=DEV, dtype=torch.int32)
    mask = torch.ones(3, size[2], dtype=torch.bool, device=DEV)
    mask[2] = False
    for m, rows in ((None, slice(1, 2)), (mask, slice(1, 3))):
        d = do.clone()
        d[rows] = float("nan")
        out, lse, lo = ops.cross_attention_fwd(q, k, v, lens, m, want_residual=True)
        got = ops.cross_attention_bwd(q, k, v, out, lse, d, lens, m, out_residual=lo)
        d[rows] = 0
        ref = ops.cross_attention_bwd(q, k, v, out, lse, d, lens, m, out_residual=lo)
        assert all(torch.equal(a, b) and bool((a[rows] == 0).all()) for a, b in zip(got, ref))


def test_more_rows_than_threads_of_a_launch():
    """2^28 rows of one problem: 16 lanes a row are more than 2^32 threads.  Only the last rows have a gradient: everything equals the small problem's."""
    from snag_amd import ops
    n, last, Lk, d = (1 << 28) + 70, 50, 3, 4
    g = torch.Generator(device=DEV).manual_seed(13)
    q = torch.empty(1, n, 1, d, device=DEV, dtype=torch.bfloat16).normal_(generator=g)
    k, v = (torch.randn(1, Lk, 1, d, generator=g, device=DEV).bfloat16() for _ in range(2))
    do = torch.zeros_like(q)
    do[:, -last:] = torch.randn(1, last, 1, d, generator=g, device=DEV).bfloat16()
    out, lse, lo = ops.cross_attention_fwd(q, k, v, want_residual=True)
    dq, dk, dv = ops.cross_attention_bwd(q, k, v, out, lse, do, out_residual=lo)
    small = q[:, -last:]
    r = attention(small, k, v, None, None, None, do[:, -last:])
    b = attention_bounds(small, k, v, None, None, None, do[:, -last:], r)
    for name, t in (("o", out[:, -last:]), ("dq", dq[:, -last:]), ("dk", dk), ("dv", dv)):
        assert bool(((t.double() - r[name]).abs() <= b[name]).all()), name
    assert bool((dq[:, :-last] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_two_streams_graph_replays_and_repeats(dtype):
    """The same bits on another stream, twice in a row, and in every replay of a captured graph with other work between; a capture while an
    eager graph of the same leaves lives is refused."""
    from snag_amd._lib import SnagHipError
    from snag_amd.cross import cross_attention
    g = torch.Generator(device=DEV).manual_seed(7)
    sets = []
    for rows, Lk in ((2, 3000), (70, 400), (8, 2000)):
        q, k, v = (torch.randn(2, L, 2, 64, generator=g, device=DEV).to(dtype).requires_grad_(True) for L in (rows, Lk, Lk))
        sets.append((q, k, v, torch.randn(2, rows, 2, 64, generator=g, device=DEV).to(dtype)))

    def all_of():
        r = []
        for q, k, v, do in sets:
            o = cross_attention(q, k, v)
            r += [o.detach(), *torch.autograd.grad(o, (q, k, v), do)]
        return r

    want = all_of()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = all_of()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = all_of()
    for i in range(4):
        for t in got:
            t.zero_()
        graph.replay()
        junk = torch.randn(1 << 20, device=DEV) * i
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), i
        assert all(torch.equal(a, b) for a, b in zip(want, all_of()))
    del junk
    alive = cross_attention(*sets[1][:3])
    with pytest.raises(SnagHipError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            cross_attention(*sets[1][:3])
    assert torch.equal(torch.autograd.grad(alive, sets[1][0], sets[1][3])[0], want[5])


def test_refusals_in_python():
    from snag_amd import ops
    q, k, v, _ = make(2, 3, 5, 4, 2, 16, torch.bfloat16)
    for bad, err in (((q.float(), k, v), TypeError), ((q, k.float(), v), TypeError), ((q, k[:, :4], v), ValueError), ((q[:1], k, v), ValueError), ((q[:, :, :3], k, v), ValueError),
                     ((q, k.transpose(2, 3).contiguous().transpose(2, 3), v), ValueError), ((q[0], k, v), ValueError)):
        with pytest.raises(err):
            ops.cross_attention_fwd(*bad)
    with pytest.raises(ValueError):
        ops.cross_attention_fwd(*make(1, 1, 1, 1, 1, 130, torch.bfloat16)[:3])
    with pytest.raises(ValueError):
        ops.cross_attention_fwd(q, k, v, kv_lens=torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(TypeError):
        ops.cross_attention_fwd(q, k, v, kv_lens=torch.zeros(2, device=DEV))
    with pytest.raises(TypeError):
        ops.cross_attention_fwd(q, k, v, key_mask=torch.zeros(2, 5, device=DEV))
    with pytest.raises(ValueError):
        ops.cross_attention_fwd(q, k, v, key_mask=torch.zeros(2, 4, dtype=torch.bool, device=DEV))
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            ops.cross_attention_fwd(q, k, v, scale=scale)
