"""Plain 64-bit statements of cross attention, the sandwich norm and the orthogonalisation, and how far a correct kernel may be from them."""
import math

import torch

f64 = torch.float64


def half_step(dtype):
    """A rounding to `dtype` is off by at most this, relative to the value ..."""
    return torch.finfo(dtype).eps / 2


def tiny_step(dtype):
    """... or by this where the value is subnormal."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def attention(q, k, v, lens=None, mask=None, scale=None, d_out=None):
    """-> {"o", "lse" (natural), "p", and with d_out "dq", "dk", "dv", "ds"}; everything in 64 bits, unseen keys never touched."""
    q, k, v = q.to(f64), k.to(f64), v.to(f64)
    B, Lq, H, d = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    scale = d ** -0.5 if scale is None else scale
    seen = torch.ones(B, Lk, dtype=torch.bool, device=q.device)
    if lens is not None:
        seen &= torch.arange(Lk, device=q.device)[None] < lens[:, None]
    if mask is not None:
        seen &= mask.bool()
    k, v = torch.where(seen[:, :, None, None], k, 0.0), torch.where(seen[:, :, None, None], v, 0.0)
    kh, vh = (t.repeat_interleave(G, dim=2).permute(0, 2, 1, 3).contiguous() for t in (k, v))      # [B, H, Lk, d]
    qh = q.permute(0, 2, 1, 3).contiguous()
    s = (qh @ kh.transpose(2, 3).contiguous()) * scale
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    lse = torch.logsumexp(s, -1) if Lk else torch.full((B, H, Lq), -math.inf, dtype=f64, device=q.device)
    p = torch.where(lse[..., None] == -math.inf, 0.0, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None]))
    o = p @ vh
    r = {"o": o.permute(0, 2, 1, 3), "lse": lse, "p": p, "seen": seen}
    if d_out is None:
        return r
    doh = d_out.to(f64).permute(0, 2, 1, 3).contiguous()
    dp = doh @ vh.transpose(2, 3).contiguous()
    delta = (doh * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    share = lambda t: t.view(B, Hkv, G, Lk, d).sum(2).permute(0, 2, 1, 3)
    r.update(dq=(ds @ kh * scale).permute(0, 2, 1, 3), dk=share(ds.transpose(2, 3).contiguous() @ qh * scale), dv=share(p.transpose(2, 3).contiguous() @ doh), ds=ds)
    return r


def attention_bounds(q, k, v, lens, mask, scale, d_out, r):
    """Elementwise bounds of a kernel that forms scores, sums and outputs in fp32 (each product and sum step off by 2^-24 of the terms'
    magnitudes, the worst case added up), rounds p and ds to the inputs' type for the second products, and rounds each output once.

      p:  the score's error, (d + 3) 2^-24 scale sum |q||k|, enters p and the row sum: twice; exp2, sum, division: (Lk + 16) 2^-24
      o:  u |o| + (u + e_p) sum p |v| (+ the second rounding's subnormal step per key)
      ds: u |ds| + e_p |ds| + p ((d + 3) 2^-24 sum |do||v| + (u + (d + 3) 2^-24) sum |do||o|)      (delta is formed from the rounded o)
    What is below the smallest normal fp32 number may become 0 (the hardware's exp2 and the matrix instruction flush): p and ds are off by up to
    2^-126 more, which p hands to ds times |dp - delta|, and so is each output.
    """
    dtype = q.dtype
    u, tiny, e = half_step(dtype), max(tiny_step(dtype), 2.0 ** -126), 2.0 ** -24
    q, k, v = (t.to(f64) for t in (q, k, v))
    B, Lq, H, d = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    scale = d ** -0.5 if scale is None else scale
    seen = r["seen"]
    k, v = torch.where(seen[:, :, None, None], k, 0.0), torch.where(seen[:, :, None, None], v, 0.0)
    kh, vh = (t.abs().repeat_interleave(G, dim=2).permute(0, 2, 1, 3).contiguous() for t in (k, v))
    qh = q.abs().permute(0, 2, 1, 3).contiguous()
    sa = qh @ kh.transpose(2, 3).contiguous() * scale
    sa = sa * seen[:, None, None]
    es = (d + 3) * e * sa
    ep = es + es.amax(-1, keepdim=True) + (Lk + 16) * e * (1 + r["lse"].abs().nan_to_num(posinf=0.0)[..., None]) if Lk else es
    p = r["p"]
    out = {"o": u * r["o"].abs() + (((u + ep) * p) @ vh + tiny * vh.sum(2, keepdim=True)).permute(0, 2, 1, 3) + tiny,
           "lse": (es.amax(-1) if Lk else 0.0) + (Lk + 16) * e * (1 + r["lse"].abs().nan_to_num(posinf=0.0))}
    if d_out is None:
        return out
    doh = d_out.to(f64).abs().permute(0, 2, 1, 3).contiguous()
    oh = r["o"].abs().permute(0, 2, 1, 3)
    rough = (d + 3) * e * (doh @ vh.transpose(2, 3).contiguous()) + (u + (d + 3) * e) * (doh * oh).sum(-1, keepdim=True) + (doh * out["o"].permute(0, 2, 1, 3)).sum(-1, keepdim=True)
    dpa = doh @ vh.transpose(2, 3).contiguous() + (doh * oh).sum(-1, keepdim=True)
    eds = (u + ep) * r["ds"].abs() + p * rough + (tiny + 2.0 ** -126 * dpa) * seen[:, None, None]
    share = lambda t: t.view(B, Hkv, G, Lk, d).sum(2).permute(0, 2, 1, 3)
    rows = G * Lq
    out["dq"] = u * r["dq"].abs() + (eds @ kh * scale + (Lk + 4) * e * (r["ds"].abs() @ kh) * scale).permute(0, 2, 1, 3) + tiny
    out["dk"] = u * r["dk"].abs() + share(eds.transpose(2, 3).contiguous() @ qh * scale + (rows + 4) * e * (r["ds"].abs().transpose(2, 3).contiguous() @ qh) * scale) + tiny
    epv = ((u + ep + (rows + 4) * e) * p + tiny * seen[:, None, None]).transpose(2, 3).contiguous()
    out["dv"] = u * r["dv"].abs() + share(epv @ doh) + tiny
    return out


def _norm(t, kind, eps):
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
    return t * r, r


def _norm_back(d, n, r, kind):
    t = d - n * (d * n).mean(-1, keepdim=True)
    return (t - d.mean(-1, keepdim=True) if kind == "layer" else t) * r


def sandwich(x, y, post_weight=None, pre_weight=None, post_bias=None, pre_bias=None, gate=None, res_scale=1.0, kind="rms", eps=1e-6, d_h=None, d_z=None):
    """-> {"h", "z"} and, when d_h or d_z is given, {"d_x", "d_y", "d_<parameter>"}; [rows, dim], in 64 bits."""
    c = lambda t, none: torch.full((1,), none, dtype=f64, device=x.device) if t is None else t.detach().to(f64)
    x, y = x.detach().to(f64), y.detach().to(f64)
    D = x.shape[-1]
    x, y = x.reshape(-1, D), y.reshape(-1, D)
    pw, qw, pb, qb = c(post_weight, 1.0), c(pre_weight, 1.0), c(post_bias, 0.0), c(pre_bias, 0.0)
    g = c(gate, 1.0)
    if gate is not None and gate.dim() == 2:
        g = g.repeat_interleave(x.shape[0] // gate.shape[0], dim=0)
    ny, ry = _norm(y, kind, eps)
    post = ny * pw + pb
    h = res_scale * x + g * post
    nh, rh = _norm(h, kind, eps)
    r = {"h": h, "z": nh * qw + qb}
    if d_h is None and d_z is None:
        return r
    dh = torch.zeros_like(h) if d_h is None else d_h.to(f64).reshape(-1, D)
    dz = torch.zeros_like(h) if d_z is None else d_z.to(f64).reshape(-1, D)
    d = dh + _norm_back(dz * qw, nh, rh, kind)
    dpost = d * g
    r.update(d_x=res_scale * d, d_y=_norm_back(dpost * pw, ny, ry, kind), d_post_weight=(dpost * ny).sum(0), d_post_bias=dpost.sum(0),
             d_pre_weight=(dz * nh).sum(0), d_pre_bias=dz.sum(0))
    if gate is not None:
        dg = d * post
        r["d_gate"] = dg.sum(0) if gate.dim() == 1 else dg.view(gate.shape[0], -1, D).sum(1)
    return r


def orthogonalized(g, steps=5, eps=1e-7):
    x = g.to(f64)
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        a = x @ x.T.contiguous()
        x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
    return x.T if tall else x


def orthogonalized_in_fp16(g, planes, steps=5, eps=1e-7):
    """The iteration in the kernel's arithmetic: operands as fp16 pairs of one scaling, `planes` 1: the leading products only with both
    diagonals kept out of them, 2: three products; sums in fp32.  Its distance from orthogonalized() is what that arithmetic costs."""
    SX, SA = 2.0 ** 14, 2.0 ** 13
    f32 = torch.float32

    def pair(t, s):
        hi = (t * s).half().to(f32)
        return hi, (t * s - hi).half().to(f32)

    def product(x, y, sx, sy):
        (a, b), (c, d) = pair(x, sx), pair(y, sy)
        r = a @ c
        if planes == 2:
            r = r + (a @ d + b @ c)
        return r / (sx * sy)

    tall = g.shape[0] > g.shape[1]
    x = (g.to(f64) / (g.to(f64).norm() + eps)).to(f32)
    x = x.T.contiguous() if tall else x
    eye = torch.eye(x.shape[0], dtype=f32, device=g.device)
    for _ in range(steps):
        hi, lo = pair(x, SX)
        x = (hi + lo) / SX
        a = product(x, x.T.contiguous(), SX, SX)
        da = a.diagonal().clone()
        r = a - a * eye
        sq = product(r, r, SA, SA)
        b = -4.7750 * a + 2.0315 * (sq + (da[:, None] + da[None]) * r + torch.diag(da * da))
        db = b.diagonal().clone()
        x = (3.4445 + db)[:, None] * x + product(b - b * eye, x, SA, SX)
    return x.T if tall else x
