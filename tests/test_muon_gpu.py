"""GPU: Newton-Schulz orthogonalisation and the Muon update against the 64-bit statement.

What the kernel's arithmetic costs is computed, not guessed: cross_reference.orthogonalized_in_fp16 states it in torch (fp16 pairs, fp32
sums), its distance from the 64-bit iteration on the same matrix is `cost`, and the kernel may be off by twice that (another order of the
fp32 sums) plus 2e-6 (the sums themselves where cost is tiny) plus half a step of the output's type."""
import math

import pytest
import torch

from cross_reference import half_step, orthogonalized, orthogonalized_in_fp16

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = [(1, 1), (1, 9), (9, 1), (3, 5), (64, 64), (128, 128), (128, 4096), (768, 128), (129, 127), (100, 300), (300, 100), (257, 513), (640, 640), (1000, 130), (384, 2000), (2, 5000)]


def gradient(r, c, dtype, seed=0, low_rank=False, scale=1e-3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    m = torch.randn(r, c, generator=g, device=DEV)
    if low_rank:
        k = max(1, min(r, c) // 8)
        m = 0.05 * m + torch.randn(r, k, generator=g, device=DEV) @ (torch.logspace(0, -2, k, device=DEV)[:, None] * torch.randn(k, c, generator=g, device=DEV))
    return (m * scale).to(dtype)


def distance(a, b):
    return float((a.detach().double() - b).norm() / b.norm())


def allowed(g, ref, dtype, steps=5):
    cost = distance(orthogonalized_in_fp16(g.float() if dtype == torch.float32 else g, 1 if dtype == torch.bfloat16 else 2, steps), ref)
    return 2 * cost + 2e-6 + half_step(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("low_rank", [False, True])
def test_list_of_all_shapes(dtype, low_rank):
    from snag_amd.optim import orthogonalize
    gs = [gradient(r, c, dtype, i, low_rank) for i, (r, c) in enumerate(SHAPES)]
    got = orthogonalize(gs)
    for g, o in zip(gs, got):
        ref = orthogonalized(g)
        assert o.dtype == dtype and o.shape == g.shape
        assert distance(o, ref) <= allowed(g, ref, dtype), (tuple(g.shape), distance(o, ref), allowed(g, ref, dtype))
    # twice: the same bits; alone or among others: another cut of the contraction, the same bounds
    assert all(torch.equal(a, b) for a, b in zip(orthogonalize(gs), got))
    for i in (0, 6, 9, 10, 12):
        ref = orthogonalized(gs[i])
        assert distance(orthogonalize(gs[i]), ref) <= allowed(gs[i], ref, dtype)
    singular = torch.linalg.svdvals(orthogonalize(gradient(200, 300, torch.float32)).double())
    assert 0.6 < float(singular.min()) and float(singular.max()) < 1.3


@pytest.mark.parametrize("steps", [1, 2, 3, 7])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps(dtype, steps):
    from snag_amd.optim import orthogonalize
    for r, c in ((150, 260), (260, 150)):
        g = gradient(r, c, dtype, 3)
        ref = orthogonalized(g, steps)
        assert distance(orthogonalize(g, steps=steps), ref) <= allowed(g, ref, dtype, steps)


def test_magnitudes_zeros_and_nan():
    from snag_amd.optim import orthogonalize
    g = gradient(130, 200, torch.float32, 4, scale=1.0)
    ref = orthogonalized(g, eps=0.0)
    for s in (1e-30, 1e-12, 1e25):                       # squares that leave fp32's range either way
        assert distance(orthogonalize(g * s, eps=0.0), ref) <= allowed(g, ref, torch.float32), s
    one = torch.zeros(300, 140, device=DEV)
    one[7, 9] = 5.0                                      # a single singular value: the largest entry X can have
    ref = orthogonalized(one)
    assert distance(orthogonalize(one), ref) <= 4e-6
    zero, bad = torch.zeros(64, 200, device=DEV), g.clone()
    bad[3, 4] = float("nan")
    a, b, c = orthogonalize([zero, bad, g])
    assert bool((a == 0).all()) and bool(b.isnan().all()) and torch.equal(c, orthogonalize(g))
    assert orthogonalize([]) == []


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_matrices_among_small_ones(dtype):
    """Shapes that take the larger tile, in one list with shapes that do not."""
    from snag_amd.optim import orthogonalize
    gs = [gradient(r, c, dtype, i) for i, (r, c) in enumerate([(200, 300), (3500, 3600), (2050, 7000), (64, 128), (5000, 2700)])]
    for g, o in zip(gs, orthogonalize(gs)):
        ref = orthogonalized(g)
        assert distance(o, ref) <= allowed(g, ref, dtype), (tuple(g.shape), distance(o, ref), allowed(g, ref, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shapes", [[(4096, 4096)], [(4700, 4200), (300, 200)], [(2900, 3000), (200, 4000), (2950, 2900)]])
def test_tiles_over_a_round(shapes, dtype):
    """More 128 x 128 tiles of the symmetric products than run at a time: the last ones are cut into ranges of the contraction."""
    from snag_amd.optim import orthogonalize
    gs = [gradient(r, c, dtype, i) for i, (r, c) in enumerate(shapes)]
    got = orthogonalize(gs)
    for g, o in zip(gs, got):
        ref = orthogonalized(g)
        assert distance(o, ref) <= allowed(g, ref, dtype), (tuple(g.shape), distance(o, ref), allowed(g, ref, dtype))
    assert all(torch.equal(a, b) for a, b in zip(orthogonalize(gs), got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nesterov, match_rms", [(True, False), (False, True)])
def test_step(dtype, nesterov, match_rms):
    """Two updates, more matrices than one launch takes (24)."""
    from snag_amd.optim import muon_step
    shapes = [(128, 700), (700, 128), (40, 40), (64, 129), (5, 3)] * 6
    ws = [gradient(r, c, dtype, 100 + i, scale=0.05) for i, (r, c) in enumerate(shapes)]
    ms = [torch.zeros(r, c, device=DEV) for r, c in shapes]
    w64, m64 = [w.double() for w in ws], [m.double() for m in ms]
    lr, mu, wd = 0.05, 0.9, 0.1
    for turn in range(2):
        gs = [gradient(r, c, dtype, 1000 * turn + i, low_rank=True) for i, (r, c) in enumerate(shapes)]
        muon_step(ws, gs, ms, lr, mu, nesterov, wd, match_rms)
        for i, (r, c) in enumerate(shapes):
            g = gs[i].double()
            m64[i] = mu * m64[i] + (1 - mu) * g
            u = (1 - mu) * g + mu * m64[i] if nesterov else m64[i]
            x = orthogonalized(u)
            s = 0.2 * math.sqrt(max(r, c)) if match_rms else math.sqrt(max(1, r / c))
            new = (1 - lr * wd) * w64[i] - lr * s * x
            assert bool(((ms[i].double() - m64[i]).abs() <= 2.0 ** -22 * (m64[i].abs() + g.abs())).all())
            # the momentum in hand is rounded to fp32: what that moves through the iteration is part of the same cost
            cost = allowed(u.to(torch.float32) if dtype == torch.float32 else u, x, torch.float32 if dtype == torch.float32 else dtype) if dtype == torch.float32 else None
            if cost is None:
                cost = 2 * distance(orthogonalized_in_fp16(u, 1), x) + 2e-6
            off = float((ws[i].double() - new).norm())
            tol = lr * s * cost * float(x.norm()) + (half_step(dtype) + 2.0 ** -22) * float(new.norm())
            assert off <= tol, (turn, i, (r, c), off, tol)
            w64[i], m64[i] = ws[i].double(), ms[i].double()


def test_in_place_graph_and_streams():
    from snag_amd import ops
    from snag_amd.optim import muon_step, orthogonalize
    gs = [gradient(r, c, torch.bfloat16, i) for i, (r, c) in enumerate([(128, 1500), (300, 200), (64, 64)])]
    want = orthogonalize(gs)
    twin = [g.clone() for g in gs]
    ops.orthogonalize(twin, twin)
    assert all(torch.equal(a, b) for a, b in zip(want, twin))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = orthogonalize(gs)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    # a captured update, replayed with other work between, walks with an eager one
    make = lambda: ([g.clone() for g in gs], [torch.zeros(g.shape, device=DEV) for g in gs])
    (w1, m1), (w2, m2) = make(), make()
    graphs = []
    for _ in range(2):                                   # two graphs of one pool share its workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            muon_step(w1, gs, m1, 0.1, weight_decay=0.01)
        graphs.append(graph)
    for i in range(4):
        graphs[i % 2].replay()
        junk = torch.randn(1 << 20, device=DEV)
        muon_step(w2, gs, m2, 0.1, weight_decay=0.01)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(w1 + m1, w2 + m2)), i
    del junk


def test_refusals_in_python():
    from snag_amd import ops
    a = torch.zeros(4, 6, device=DEV)
    for gs, err in (([a[0]], ValueError), ([a.t()], ValueError), ([a, a.bfloat16()], TypeError), ([a.double()], TypeError), ([torch.zeros(0, 3, device=DEV)], ValueError)):
        with pytest.raises(err):
            ops.orthogonalize(gs)
    with pytest.raises(ValueError):
        ops.orthogonalize([a], steps=0)
    b = a.clone()
    for args, err in ((([a], [a, a], [b]), ValueError), (([a], [a], [b.bfloat16()]), TypeError), (([a], [a.bfloat16()], [b]), TypeError), (([a], [a[:3]], [b]), ValueError),
                      (([a, a], [a, a], [b, b.clone()]), ValueError), (([a], [b], [a]), ValueError), (([a], [a], [b]), ValueError), (([a[:2], a[1:3]], [b[:2], b[:2]], [b[2:], b.clone()[:2]]), ValueError)):
        with pytest.raises(err):
            ops.muon_step(*args, lr=0.1)
    # written in place: a graph that saved the old values refuses to run on the new ones
    w = a.clone().requires_grad_(True)
    y = (w * w).sum()
    ops.muon_step([w.detach()], [torch.ones_like(a)], [b], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_resumed_optimizer_goes_on_bit_for_bit(dtype):
    from snag_amd.optim import Muon
    g = torch.Generator(device=DEV).manual_seed(15)
    grads = [torch.randn(40, 70, generator=g, device=DEV).to(dtype) for _ in range(4)]
    w = torch.nn.Parameter(torch.randn(40, 70, generator=g, device=DEV).to(dtype))
    opt = Muon([w], lr=0.1)
    for d in grads[:2]:
        w.grad = d
        opt.step()
    copy = torch.nn.Parameter(w.detach().clone())
    again = Muon([copy], lr=0.1)
    again.load_state_dict({"state": {i: {k: t.clone() for k, t in s.items()} for i, s in opt.state_dict()["state"].items()}, "param_groups": opt.state_dict()["param_groups"]})
    for p, o in ((w, opt), (copy, again)):
        for d in grads[2:]:
            p.grad = d
            o.step()
    assert torch.equal(w, copy)


def test_a_block_trained_by_the_optimizer():
    """The operators together, as they are used: a cross-modal layer over ragged states, its gradients against the 64-bit statement, and
    updates of its matrices (Muon) and vectors (AdamW) by one optimiser."""
    import torch.nn.functional as F
    from cross_reference import attention, sandwich
    from snag_amd.cross import CrossModalLayer
    from snag_amd.optim import Muon
    torch.manual_seed(0)
    N, M, L, D, S = 37, 3, 21, 64, 48
    layer = CrossModalLayer(D, 4, state_dim=S, kv_heads=2, intermediate_size=96, kind="layer").to(DEV)
    x, states = torch.randn(N, M, D, device=DEV), torch.randn(N, L, S, device=DEV)
    lens = torch.randint(0, L + 1, (N,), device=DEV, dtype=torch.int32)
    lens[0] = 0
    dh, dz = torch.randn(N, M, D, device=DEV), torch.randn(N, M, D, device=DEV)
    h, z = layer(x, states, lens)
    ((h * dh).sum() + (z * dz).sum()).backward()
    # the statement, differentiated in 64 bits
    p = {n: t.detach().double().requires_grad_(True) for n, t in layer.named_parameters()}

    def norm(xx, yy, pre):
        ln = lambda t: F.layer_norm(t, (D,), eps=1e-6)
        hh = xx + p[pre + ".gate"] * (ln(yy) * p[pre + ".post_weight"])
        return hh, ln(hh) * p[pre + ".pre_weight"]

    lin = lambda t, n: t @ p[n + ".weight"].T + p[n + ".bias"]
    q = lin(x.double(), "query").view(N, M, 4, 16)
    k, v = (lin(states.double(), n).view(N, L, 2, 16).repeat_interleave(2, 2) for n in ("key", "value"))
    s = torch.einsum("nmhd,nlhd->nhml", q, k) / 4
    s = s.masked_fill(torch.arange(L, device=DEV)[None, None, None] >= lens[:, None, None, None], -float("inf"))
    a = torch.einsum("nhml,nlhd->nmhd", torch.softmax(s, -1).nan_to_num(0.0), v).reshape(N, M, D)
    hh, zz = norm(x.double(), lin(a, "output"), "attention_norm")
    f = (zz @ p["feed_forward.l1.weight"].T).relu() @ p["feed_forward.l2.weight"].T
    hh, zz = norm(hh, f, "feed_forward_norm")
    assert distance(h, hh) < 1e-5 and distance(z, zz) < 1e-5
    grads = torch.autograd.grad((hh * dh).sum() + (zz * dz).sum(), list(p.values()), allow_unused=True)
    for (n, t), g in zip(layer.named_parameters(), grads):
        if n == "key.bias":
            # a constant added to every key moves all scores of a row alike and no probability: sum_s ds = 0, so this gradient is 0 and what is
            # left of it is the rounding of sums as large as the key weight's
            assert float(g.norm()) < 1e-12 and float(t.grad.norm()) < 1e-5 * float(layer.key.weight.grad.norm())
            continue
        assert distance(t.grad, g) < 1e-4, n             # fp32 chains of four products of up to 96 terms, a ReLU kink may flip
    matrices = [t for t in layer.parameters() if t.dim() == 2]
    vectors = [t for t in layer.parameters() if t.dim() != 2]
    opt = Muon([{"params": matrices}, {"params": vectors, "muon": False, "lr": 1e-3}], lr=0.02)
    before = {n: t.detach().clone() for n, t in layer.named_parameters()}
    for _ in range(3):
        opt.step()
        opt.zero_grad()
        h, z = layer(x, states, lens)
        (h.square().mean() + z.square().mean()).backward()
    for n, t in layer.named_parameters():
        assert bool(torch.isfinite(t).all()) and not torch.equal(t, before[n]), n
    state = opt.state_dict()
    again = Muon([{"params": matrices}, {"params": vectors, "muon": False, "lr": 1e-3}], lr=0.02)
    again.load_state_dict(state)
    assert all(torch.equal(again.state[t]["momentum_buffer"], opt.state[t]["momentum_buffer"]) for t in matrices)
