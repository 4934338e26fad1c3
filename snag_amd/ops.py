"""Thin, checked Python wrappers over the C ABI: tensors in, tensors out, no arithmetic here.

Shape/dtype/contiguity errors are raised in Python before the call, mirroring the reference's
assert/exception convention (SURVEY.md par. 8b "Errors").
"""
import ctypes
import functools

import torch

from . import _lib
from ._lib import call, ptr, stream

f32 = torch.float32


def _chk(t, name, dtype=f32, ndim=None):
    if not torch.is_tensor(t):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise _lib.SnagHipError(f"{name}: tensor is on {t.device}; snag_amd kernels run on the GPU only (no CPU fallback)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name}: expected dtype {dtype}, got {t.dtype}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name}: expected {ndim} dims, got shape {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: tensor must be contiguous")
    return t


def _idx(t, name, ndim):
    if not torch.is_tensor(t) or t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: expected an int32/int64 tensor")
    return _chk(t, name, dtype=None, ndim=ndim)


def _idx_group(h, r, t, neg_t):
    _idx(h, "h", 1), _idx(r, "r", 1), _idx(t, "t", 1)
    B = h.shape[0]
    if r.shape[0] != B or t.shape[0] != B:
        raise ValueError(f"h, r, t must have equal length, got {B}, {r.shape[0]}, {t.shape[0]}")
    dt = h.dtype
    if r.dtype != dt or t.dtype != dt:
        raise TypeError("h, r, t must share one index dtype")
    K = 0
    if neg_t is not None:
        _idx(neg_t, "neg_t", 2)
        if neg_t.shape[0] != B or neg_t.dtype != dt:
            raise ValueError(f"neg_t must be [{B}, K] of dtype {dt}, got {tuple(neg_t.shape)} {neg_t.dtype}")
        K = neg_t.shape[1]
    return B, K, (4 if dt == torch.int32 else 8)


def _rows(t, name):
    """2-D fp32 CUDA tensor with unit inner stride (row stride free: lets a [N, M, D] slot be used in place)."""
    if not (torch.is_tensor(t) and t.dim() == 2 and t.dtype == f32 and t.stride(1) == 1):
        raise ValueError(f"{name}: expected a 2-D fp32 tensor with unit inner stride")
    if not t.is_cuda:
        raise _lib.SnagHipError(f"{name}: tensor is on {t.device}; snag_amd kernels run on the GPU only (no CPU fallback)")
    return t


def _quads(entry, **tensors):
    """The entry moves rows as float4: every base pointer 16-byte aligned, every row stride a multiple of four floats (what the C ABI
    itself refuses with SNAG_ERR_UNSUPPORTED; checked here for the readable message)."""
    for name, t in tensors.items():
        if t.numel() and (t.data_ptr() % 16 or (t.dim() == 2 and t.stride(0) % 4)):
            raise ValueError(f"{entry}: {name} must be 16-byte aligned with a row stride that is a multiple of 4 floats "
                             f"(data_ptr % 16 = {t.data_ptr() % 16}, strides {tuple(t.stride())})")


def score_margin_fwd(ent, rel, h, r, t, neg_t, margin, want_loss=True):
    """-> pos [B], neg [B,K], loss_part [B] (or None).  C ABI: snag_score_margin_fwd."""
    _rows(ent, "ent"), _chk(rel, "rel", ndim=2)
    if ent.shape[1] != rel.shape[1]:
        raise ValueError(f"ent dim {ent.shape[1]} != rel dim {rel.shape[1]}")
    B, K, ib = _idx_group(h, r, t, neg_t)
    pos = torch.empty(B, device=ent.device, dtype=f32)
    neg = torch.empty(B, K, device=ent.device, dtype=f32)
    loss_part = torch.empty(B, device=ent.device, dtype=f32) if want_loss else None
    call("snag_score_margin_fwd", ptr(ent), ent.stride(0), ent.shape[0], ptr(rel), rel.shape[0], ent.shape[1],
         ptr(h), ptr(r), ptr(t), ptr(neg_t), ib, B, K, float(margin), ptr(pos), ptr(neg), ptr(loss_part), stream())
    return pos, neg, loss_part


def score_margin_fwd_bf16(ent, rel, h, r, t, neg_t, margin, want_loss=True):
    """bf16 tables -> fp32 scores.  C ABI: snag_score_margin_fwd_bf16."""
    for x, nm in ((ent, "ent"), (rel, "rel")):
        if not (torch.is_tensor(x) and x.is_cuda and x.dtype == torch.bfloat16 and x.dim() == 2 and x.stride(1) == 1):
            raise ValueError(f"{nm}: expected a 2-D bfloat16 CUDA tensor with unit inner stride")
    if not rel.is_contiguous():
        raise ValueError("rel must be contiguous")
    B, K, ib = _idx_group(h, r, t, neg_t)
    pos = torch.empty(B, device=ent.device, dtype=f32)
    neg = torch.empty(B, K, device=ent.device, dtype=f32)
    loss_part = torch.empty(B, device=ent.device, dtype=f32) if want_loss else None
    call("snag_score_margin_fwd_bf16", ptr(ent), ent.stride(0), ent.shape[0], ptr(rel), rel.shape[0], ent.shape[1],
         ptr(h), ptr(r), ptr(t), ptr(neg_t), ib, B, K, float(margin), ptr(pos), ptr(neg), ptr(loss_part), stream())
    return pos, neg, loss_part


def score_margin_bwd(ent, rel, h, r, t, neg_t, margin, grad_scale=1.0, dpos=None, dneg=None, d_ent=None, d_rel=None):
    """Accumulates into d_ent/d_rel (allocated zeroed when None).  C ABI: snag_score_margin_bwd."""
    _rows(ent, "ent"), _chk(rel, "rel", ndim=2)
    B, K, ib = _idx_group(h, r, t, neg_t)
    if dpos is not None:
        _chk(dpos, "dpos", ndim=1)
        if dpos.shape[0] != B:
            raise ValueError("dpos must be [B]")
    if dneg is not None:
        _chk(dneg, "dneg", ndim=2)
        if tuple(dneg.shape) != (B, K):
            raise ValueError("dneg must be [B, K]")
    if d_ent is None:
        d_ent = torch.zeros(ent.shape, device=ent.device, dtype=f32)
    if d_rel is None:
        d_rel = torch.zeros_like(rel)
    _rows(d_ent, "d_ent"), _chk(d_rel, "d_rel", ndim=2)
    if d_ent.shape != ent.shape or d_rel.shape != rel.shape:
        raise ValueError("gradient buffers must match the table shapes")
    call("snag_score_margin_bwd", ptr(ent), ent.stride(0), ent.shape[0], ptr(rel), rel.shape[0], ent.shape[1],
         ptr(h), ptr(r), ptr(t), ptr(neg_t), ib, B, K, float(margin), float(grad_scale),
         ptr(dpos), ptr(dneg), ptr(d_ent), d_ent.stride(0), ptr(d_rel), stream())
    return d_ent, d_rel


_TICKETS = {}


def _ticket(device):
    """SNAG_SCORE_TICKET_WORDS zeroed uint32 per device for the fused scorer's last-block reduction (the kernel leaves it zero again)."""
    key = (device.type, device.index, stream())          # per stream: two streams' launches must not share the ticket words
    if key not in _TICKETS:
        _TICKETS[key] = torch.zeros(_lib.SCORE_TICKET_WORDS, device=device, dtype=torch.int32)
    return _TICKETS[key]


def score_margin_fwd_bwd(ent, rel, h, r, t, neg_t, margin, grad_scale=1.0, d_ent=None, d_rel=None, want_loss=True):
    """Hinge scorer, forward and backward in one launch -> (loss 0-dim or None, pos [B], neg [B,K], loss_part [B], d_ent, d_rel).
    Accumulates into d_ent / d_rel (allocated zeroed when None).  C ABI: snag_score_margin_fwd_bwd."""
    _rows(ent, "ent"), _chk(rel, "rel", ndim=2)
    if ent.shape[1] != rel.shape[1]:
        raise ValueError(f"ent dim {ent.shape[1]} != rel dim {rel.shape[1]}")
    if neg_t is None:
        raise ValueError("score_margin_fwd_bwd needs explicit negative tails")
    B, K, ib = _idx_group(h, r, t, neg_t)
    if d_ent is None:
        d_ent = torch.zeros(ent.shape, device=ent.device, dtype=f32)
    if d_rel is None:
        d_rel = torch.zeros_like(rel)
    _rows(d_ent, "d_ent"), _chk(d_rel, "d_rel", ndim=2)
    if d_ent.shape != ent.shape or d_rel.shape != rel.shape:
        raise ValueError("gradient buffers must match the table shapes")
    pos = torch.empty(B, device=ent.device, dtype=f32)
    neg = torch.empty(B, K, device=ent.device, dtype=f32)
    loss_part = torch.empty(B, device=ent.device, dtype=f32)
    loss = torch.empty((), device=ent.device, dtype=f32) if want_loss else None
    call("snag_score_margin_fwd_bwd", ptr(ent), ent.stride(0), ent.shape[0], ptr(rel), rel.shape[0], ent.shape[1],
         ptr(h), ptr(r), ptr(t), ptr(neg_t), ib, B, K, float(margin), float(grad_scale), ptr(pos), ptr(neg), ptr(loss_part),
         ptr(loss), ptr(_ticket(ent.device)) if want_loss else None, ptr(d_ent), d_ent.stride(0), ptr(d_rel), stream())
    return loss, pos, neg, loss_part, d_ent, d_rel


_SEG_WORK = {}           # at most _SEG_WORK_MAX workspaces, least recently used dropped (ragged batch sizes would otherwise keep one each)
_SEG_WORK_MAX = 4


def score_margin_fwd_bwd_seg(ent, rel, h, r, t, neg_t, margin, grad_scale=1.0, d_ent=None, d_rel=None, write_untouched=True):
    """Hinge scorer, forward and backward WITHOUT float atomics (per-triple pass + per-destination pass, bit-reproducible)
    -> (loss, pos, neg, loss_part, d_ent, d_rel); d_ent / d_rel are overwritten.  C ABI: snag_score_margin_fwd_bwd_seg."""
    _rows(ent, "ent"), _chk(rel, "rel", ndim=2)
    if ent.shape[1] != rel.shape[1]:
        raise ValueError(f"ent dim {ent.shape[1]} != rel dim {rel.shape[1]}")
    if neg_t is None:
        raise ValueError("score_margin_fwd_bwd_seg needs explicit negative tails")
    B, K, ib = _idx_group(h, r, t, neg_t)
    if d_ent is None:
        d_ent = torch.empty(ent.shape, device=ent.device, dtype=f32) if write_untouched else torch.zeros(ent.shape, device=ent.device, dtype=f32)
    if d_rel is None:
        d_rel = torch.empty_like(rel) if write_untouched else torch.zeros_like(rel)
    _rows(d_ent, "d_ent"), _chk(d_rel, "d_rel", ndim=2)
    if d_ent.shape != ent.shape or d_rel.shape != rel.shape:
        raise ValueError("gradient buffers must match the table shapes")
    N, R, D = ent.shape[0], rel.shape[0], ent.shape[1]
    nbytes = _lib.load().snag_score_seg_work_bytes(N, R, B, K, D)
    # The workspace and the ticket words belong to ONE stream at a time (the launches hand their header phase and counters to each
    # other in stream order): they are keyed by the stream as well, so two streams never share them.
    key = (ent.device.type, ent.device.index, stream(), N, R, B, K, D)
    if key not in _SEG_WORK:                     # zeroed ONCE; every launch leaves it ready for the next
        while len(_SEG_WORK) >= _SEG_WORK_MAX:
            _SEG_WORK.pop(next(iter(_SEG_WORK)))
        _SEG_WORK[key] = torch.zeros((nbytes + 255) // 256 * 256, device=ent.device, dtype=torch.uint8)
    work = _SEG_WORK[key] = _SEG_WORK.pop(key)   # (re-inserted: most recently used last)
    pos = torch.empty(B, device=ent.device, dtype=f32)
    neg = torch.empty(B, K, device=ent.device, dtype=f32)
    loss_part = torch.empty(B, device=ent.device, dtype=f32)
    loss = torch.empty((), device=ent.device, dtype=f32)
    call("snag_score_margin_fwd_bwd_seg", ptr(ent), ent.stride(0), N, ptr(rel), R, D, ptr(h), ptr(r), ptr(t), ptr(neg_t), ib, B, K, float(margin),
         float(grad_scale), ptr(pos), ptr(neg), ptr(loss_part), ptr(loss), ptr(_ticket(ent.device)), ptr(d_ent), d_ent.stride(0), ptr(d_rel),
         int(write_untouched), ptr(work), work.numel(), stream())
    return loss, pos, neg, loss_part, d_ent, d_rel


def score_margin_fwd_bwd_seg_ln(t_pre, gamma, beta, rel, h, r, t, neg_t, margin, grad_scale=1.0, keep=None, keep_p=0.0, eps=1e-12):
    """The segmented hinge scorer on the table ent = LayerNorm(t_pre) (formed here with torch, as the Mformer's read-out rows are by the
    fusion forward), its entity gradient carried through the LayerNorm inside the per-destination pass:
    -> the 10-tuple (loss, pos, neg, dt [N, D], dtm or None, dgamma, dbeta, dcol [D] (column sums of dtm-or-dt), d_rel, ent [N, D] (the
    LayerNorm output the scorer gathered)).
    C ABI: snag_score_margin_fwd_bwd_seg_ln (the partial slab is reduced here with torch, in slab order)."""
    _rows(t_pre, "t_pre"), _chk(rel, "rel", ndim=2)
    N, D = t_pre.shape
    R = rel.shape[0]
    mean = t_pre.mean(dim=1, keepdim=True)
    var = ((t_pre - mean) ** 2).mean(dim=1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    ent = ((t_pre - mean) * rstd * gamma + beta).contiguous()
    stats = torch.cat([mean, rstd], dim=1).contiguous()
    B, K, ib = _idx_group(h, r, t, neg_t)
    nbytes = _lib.load().snag_score_seg_work_bytes(N, R, B, K, D)
    work = torch.zeros((nbytes + 255) // 256 * 256, device=ent.device, dtype=torch.uint8)
    pos, neg = torch.empty(B, device=ent.device, dtype=f32), torch.empty(B, K, device=ent.device, dtype=f32)
    loss_part, loss = torch.empty(B, device=ent.device, dtype=f32), torch.empty((), device=ent.device, dtype=f32)
    d_rel = torch.empty_like(rel)
    nblk = (N + 15) // 16
    dt = torch.empty(N, D, device=ent.device, dtype=f32)
    dtm = torch.empty(N, D, device=ent.device, dtype=f32) if keep is not None else None
    part = torch.zeros(nblk, 3, D, device=ent.device, dtype=f32)
    tl = _lib.LnBwdTail()
    tl.t, tl.stats, tl.gamma = ptr(t_pre), ptr(stats), ptr(gamma)
    if keep is not None:
        _chk(keep, "keep", dtype=torch.uint8, ndim=2)
        tl.keep, tl.keep_ld, tl.keep_scale, tl.dtm = ptr(keep), keep.stride(0), 1.0 / (1.0 - keep_p), ptr(dtm)
    tl.dt, tl.part = ptr(dt), ptr(part)
    import ctypes
    call("snag_score_margin_fwd_bwd_seg_ln", ptr(ent), N, ptr(rel), R, D, ptr(h), ptr(r), ptr(t), ptr(neg_t), ib, B, K, float(margin), float(grad_scale),
         ptr(pos), ptr(neg), ptr(loss_part), ptr(loss), ptr(d_rel), ptr(work), work.numel(), ctypes.byref(tl), stream())
    sums = part.sum(dim=0)
    return loss, pos, neg, dt, dtm, sums[0], sums[1], sums[2], d_rel, ent


_TOUCHED_WORK = {}


def score_margin_fwd_bwd_touched(ent, rel, h, r, t, neg_t, margin, grad_scale=1.0, d_ent=None, d_rel=None):
    """The segmented hinge scorer for tables far larger than a batch's footprint: pass B walks the compact list of destinations that
    received an entry instead of every counter.  Only touched rows of d_ent are written -- OVERWRITTEN, not accumulated into (allocated zeroed
    when None; the caller keeps the untouched rows zero) -- and EVERY row of d_rel is overwritten (zeros for relations the batch does not
    name): a d_rel holding gradients of an earlier call loses them (since SNAG_ABI_VERSION 2; the earlier form accumulated).  fp32 or
    bfloat16 tables.  -> (loss, pos, neg, loss_part, d_ent, d_rel).  C ABI: snag_score_margin_fwd_bwd_touched(_bf16)."""
    bf16 = ent.dtype == torch.bfloat16
    for x, nm in ((ent, "ent"), (rel, "rel")):
        if not (torch.is_tensor(x) and x.is_cuda and x.dtype == (torch.bfloat16 if bf16 else f32) and x.dim() == 2 and x.stride(1) == 1):
            raise ValueError(f"{nm}: expected a 2-D {'bfloat16' if bf16 else 'fp32'} CUDA tensor with unit inner stride")
    if not rel.is_contiguous() or ent.shape[1] != rel.shape[1]:
        raise ValueError("rel must be contiguous and as wide as ent")
    if neg_t is None:
        raise ValueError("score_margin_fwd_bwd_touched needs explicit negative tails")
    B, K, ib = _idx_group(h, r, t, neg_t)
    N, R, D = ent.shape[0], rel.shape[0], ent.shape[1]
    if d_ent is None:
        d_ent = torch.zeros(N, D, device=ent.device, dtype=f32)
    if d_rel is None:
        d_rel = torch.zeros(R, D, device=ent.device, dtype=f32)
    _rows(d_ent, "d_ent"), _chk(d_rel, "d_rel", ndim=2)
    if tuple(d_ent.shape) != (N, D) or tuple(d_rel.shape) != (R, D):
        raise ValueError("gradient buffers must match the table shapes")
    nbytes = _lib.load().snag_score_touched_work_bytes(N, R, B, K, D)
    key = (ent.device.type, ent.device.index, stream(), N, R, B, K, D)
    if key not in _TOUCHED_WORK:                 # zeroed ONCE; every launch leaves it ready for the next
        while len(_TOUCHED_WORK) >= _SEG_WORK_MAX:
            _TOUCHED_WORK.pop(next(iter(_TOUCHED_WORK)))
        _TOUCHED_WORK[key] = torch.zeros((nbytes + 255) // 256 * 256, device=ent.device, dtype=torch.uint8)
    work = _TOUCHED_WORK[key] = _TOUCHED_WORK.pop(key)
    pos = torch.empty(B, device=ent.device, dtype=f32)
    neg = torch.empty(B, K, device=ent.device, dtype=f32)
    loss_part = torch.empty(B, device=ent.device, dtype=f32)
    loss = torch.empty((), device=ent.device, dtype=f32)
    call("snag_score_margin_fwd_bwd_touched_bf16" if bf16 else "snag_score_margin_fwd_bwd_touched", ptr(ent), ent.stride(0), N, ptr(rel), R, D, ptr(h), ptr(r),
         ptr(t), ptr(neg_t), ib, B, K, float(margin), float(grad_scale), ptr(pos), ptr(neg), ptr(loss_part), ptr(loss), ptr(d_ent), d_ent.stride(0),
         ptr(d_rel), ptr(work), work.numel(), stream())
    return loss, pos, neg, loss_part, d_ent, d_rel


def reduce_sum(x):
    """Deterministic sum of a float tensor -> 0-dim tensor.  C ABI: snag_reduce_sum."""
    _chk(x, "x")
    out = torch.empty((), device=x.device, dtype=f32)
    call("snag_reduce_sum", ptr(x), x.numel(), ptr(out), stream())
    return out


ACT = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_grad": 3, "relu_grad": 4}


def gram(z, alpha=1.0, out=None):
    """S = alpha * Z Z^T, symmetric bit for bit, upper-triangle tiles only (C ABI: snag_gram_f32)."""
    if not (torch.is_tensor(z) and z.is_cuda and z.dtype == f32 and z.dim() == 2 and z.stride(1) == 1):
        raise ValueError("gram: z must be a 2-D fp32 CUDA tensor with unit inner stride")
    n, k = z.shape
    if out is None:
        out = torch.empty(n, n, device=z.device, dtype=f32)
    if tuple(out.shape) != (n, n) or out.stride(1) != 1 or out.dtype != f32:
        raise ValueError("gram: out has the wrong shape")
    call("snag_gram_f32", ptr(z), z.stride(0), n, k, float(alpha), ptr(out), out.stride(0), stream())
    return out


def gemm(a, b, *, a_kcontig=True, b_kcontig=True, bias=None, alpha=1.0, act=None, want_pre_act=False,
         keep_mask=None, keep_p=0.0, add1=None, add2=None, out=None, accumulate=False, splitk=True, aux=None, c_transposed=False):
    """C = add1 + add2 + keep * act(alpha * A.B + bias)   (C ABI: snag_gemm_f32; fp32 via split-bf16 MFMA).

    a: [M,K] if a_kcontig else [K,M];  b: [N,K] if b_kcontig else [K,N]  (2-D, last dim contiguous,
    row stride free).  Returns C [M,N] (and the pre-activation when want_pre_act).
    """
    for t, nm in ((a, "a"), (b, "b")):
        if not (torch.is_tensor(t) and t.is_cuda and t.dtype == f32 and t.dim() == 2 and t.stride(1) == 1):
            raise ValueError(f"gemm: {nm} must be a 2-D fp32 CUDA tensor with unit inner stride")
    M, K = a.shape if a_kcontig else (a.shape[1], a.shape[0])
    N, Kb = (b.shape if b_kcontig else (b.shape[1], b.shape[0]))
    if K != Kb:
        raise ValueError(f"gemm: inner sizes differ ({K} vs {Kb})")
    oshape = (N, M) if c_transposed else (M, N)
    if out is None:
        out = torch.empty(oshape, device=a.device, dtype=f32)
    if tuple(out.shape) != oshape or out.stride(1) != 1:
        raise ValueError("gemm: out has the wrong shape")
    d = _lib.GemmDesc()
    d.M, d.N, d.K = M, N, K
    d.a_kcontig, d.b_kcontig = int(a_kcontig), int(b_kcontig)
    d.c_transposed = int(c_transposed)
    d.A, d.lda = ptr(a), a.stride(0)
    d.B, d.ldb = ptr(b), b.stride(0)
    d.C, d.ldc = ptr(out), out.stride(0)
    d.bias = ptr(_chk(bias, "bias", ndim=1)) if bias is not None else None
    d.alpha = float(alpha)
    d.act = ACT[act]
    pre = None
    if want_pre_act:
        pre = torch.empty_strided((M, N), (out.stride(0), 1), device=a.device, dtype=f32)
        d.pre_act = ptr(pre)
    if keep_mask is not None:
        _chk(keep_mask, "keep_mask", dtype=torch.uint8, ndim=2)
        if tuple(keep_mask.shape) != (M, N):
            raise ValueError("gemm: keep_mask must be [M,N]")
        d.keep_mask, d.keep_scale = ptr(keep_mask), 1.0 / (1.0 - keep_p)
    for nm, t in (("add1", add1), ("add2", add2)):
        if t is not None:
            if tuple(t.shape) != (M, N) or t.stride(1) != 1 or t.dtype != f32:
                raise ValueError(f"gemm: {nm} must be [M,N] fp32")
            setattr(d, nm, ptr(t))
            setattr(d, "ld" + nm[-1], t.stride(0))
    d.accumulate = int(accumulate)
    if aux is not None:
        if tuple(aux.shape) != (M, N) or aux.stride(1) != 1 or aux.dtype != f32:
            raise ValueError("gemm: aux must be [M,N] fp32")
        d.aux, d.ldaux = ptr(aux), aux.stride(0)
    ws = None
    if splitk:
        nws = _lib.load().snag_gemm_workspace_floats(M, N, K)
        if nws:
            ws = torch.empty(nws, device=a.device, dtype=f32)
            d.workspace, d.workspace_floats = ptr(ws), nws
    import ctypes
    call("snag_gemm_f32", ctypes.byref(d), stream())
    return (out, pre) if want_pre_act else out


# ---- a6 noise / statistics ------------------------------------------------------------------------
def colstats(x, exclude=None, n_valid=None, want_std=True):
    """Per-column mean and unbiased std over rows with exclude == 0.  C ABI: snag_colstats."""
    _chk(x, "x", ndim=2)
    R, C = x.shape
    if exclude is not None:
        _chk(exclude, "exclude", dtype=torch.uint8, ndim=1)
        if n_valid is None:
            n_valid = R - int(exclude.sum().item())
    elif n_valid is None:
        n_valid = R
    mean = torch.empty(C, device=x.device, dtype=f32)
    std = torch.empty(C, device=x.device, dtype=f32) if want_std else None
    work = torch.empty(_lib.load().snag_colstats_work_floats(C), device=x.device, dtype=f32)
    call("snag_colstats", ptr(x), R, C, ptr(exclude), int(n_valid), ptr(mean), ptr(std), ptr(work), stream())
    return mean, std


def noise_apply(x, mean, std, row_mask, mask_ratio, z=None, sel_index=None, seed=0, out=None):
    """Row-level Gaussian noise injection.  C ABI: snag_noise_apply."""
    _chk(x, "x", ndim=2), _chk(mean, "mean", ndim=1), _chk(std, "std", ndim=1)
    _chk(row_mask, "row_mask", dtype=torch.uint8, ndim=1)
    N, F = x.shape
    if row_mask.shape[0] != N or mean.shape[0] != F or std.shape[0] != F:
        raise ValueError("noise_apply: shape mismatch")
    if z is not None:
        _chk(z, "z", ndim=2)
        _chk(sel_index, "sel_index", dtype=torch.int32, ndim=1)
    if out is None:
        out = torch.empty_like(x)
    call("snag_noise_apply", ptr(x), N, F, ptr(mean), ptr(std), ptr(row_mask), ptr(sel_index), ptr(z),
         int(seed), float(mask_ratio), ptr(out), stream())
    return out


def dropout_keep_mask(shape, p, seed, device="cuda", tick=None, out=None):
    """uint8 keep mask (u >= p) from Philox(seed [+ device tick]).  C ABI: snag_dropout_keep_mask."""
    if out is None:
        out = torch.empty(shape, device=device, dtype=torch.uint8)
    call("snag_dropout_keep_mask", int(seed), ptr(tick), out.numel(), float(p), ptr(out), stream())
    return out


def gaussian_fill(mean, std, N, seed):
    """[N, F] tensor mean + std * z.  C ABI: snag_gaussian_fill."""
    _chk(mean, "mean", ndim=1), _chk(std, "std", ndim=1)
    out = torch.empty(N, mean.shape[0], device=mean.device, dtype=f32)
    call("snag_gaussian_fill", int(seed), N, mean.shape[0], ptr(mean), ptr(std), ptr(out), stream())
    return out


def colsum(x, out=None, accumulate=False):
    """out[c] = sum_r x[r, c] for a 2-D tensor with free row stride.  C ABI: snag_colsum."""
    _rows(x, "x")
    R, C = x.shape
    if out is None:
        out = torch.empty(C, device=x.device, dtype=f32)
    work = torch.empty(256 * C, device=x.device, dtype=f32)
    call("snag_colsum", ptr(x), R, C, x.stride(0), ptr(out), int(accumulate), ptr(work), stream())
    return out


def pack_tokens(embs, g_slot=-1, noise=None, noise_mask=None, mask_ratio=0.0, out=None):
    """torch.stack(embs, dim=1) (+ entity-noise blend in slot g_slot).  C ABI: snag_pack_tokens."""
    import ctypes
    M = len(embs)
    for i, e in enumerate(embs):
        _chk(e, f"embs[{i}]", ndim=2)
    N, D = embs[0].shape
    if out is None:
        out = torch.empty(N, M, D, device=embs[0].device, dtype=f32)
    arr = (ctypes.c_void_p * M)(*[e.data_ptr() for e in embs])
    if noise is not None:
        _chk(noise, "noise", ndim=2), _chk(noise_mask, "noise_mask", dtype=torch.uint8, ndim=1)
    call("snag_pack_tokens", arr, M, N, D, g_slot % M if M else 0, ptr(noise), ptr(noise_mask), float(mask_ratio) * 0.5,
         ptr(out), stream())
    return out


def atten_weight_fwd(x, a, out=None):
    """README joint_way "atten_weight": x [rows, M, D] tokens, a [D] -> (out [rows, D] = sum_m softmax_m(relu(x_m . a)) x_m, aw [rows, 2 M] = the
    weights and pre-activations the backward reads).  C ABI: snag_atten_weight_fwd (arithmetic: model/EVA_tools.py:190-232)."""
    _chk(x, "x", ndim=3), _chk(a, "a", ndim=1)
    rows, M, D = x.shape
    if a.shape[0] != D:
        raise ValueError(f"a has {a.shape[0]} entries, the tokens are {D} wide")
    if out is None:
        out = torch.empty(rows, D, device=x.device, dtype=f32)
    _rows(out, "out")
    if D % 4 == 0:            # (otherwise the C ABI refuses the shape itself)
        _quads("atten_weight_fwd", x=x, a=a, out=out)
    aw = torch.empty(rows, 2 * M, device=x.device, dtype=f32)
    call("snag_atten_weight_fwd", ptr(x), rows, M, D, ptr(a), ptr(out), out.stride(0), ptr(aw), stream())
    return out, aw


def atten_weight_bwd(x, a, aw, d_out, d_x=None, d_a=None, accumulate_da=False):
    """-> (d_x [rows, M, D], d_a [D]).  C ABI: snag_atten_weight_bwd."""
    _chk(x, "x", ndim=3), _chk(a, "a", ndim=1), _chk(aw, "aw", ndim=2), _rows(d_out, "d_out")
    rows, M, D = x.shape
    if tuple(aw.shape) != (rows, 2 * M) or tuple(d_out.shape) != (rows, D):
        raise ValueError(f"aw must be [{rows}, {2 * M}] and d_out [{rows}, {D}], got {tuple(aw.shape)}, {tuple(d_out.shape)}")
    d_x = torch.empty_like(x) if d_x is None else _chk(d_x, "d_x", ndim=3)
    d_a = torch.zeros(D, device=x.device, dtype=f32) if d_a is None else _chk(d_a, "d_a", ndim=1)
    if D % 4 == 0:
        _quads("atten_weight_bwd", x=x, a=a, d_out=d_out, d_x=d_x)
    work = torch.empty(max(1, _lib.load().snag_atten_weight_work_floats(D)), device=x.device, dtype=f32)
    call("snag_atten_weight_bwd", ptr(x), rows, M, D, ptr(a), ptr(aw), ptr(d_out), d_out.stride(0), ptr(d_x), ptr(d_a), int(accumulate_da), ptr(work), stream())
    return d_x, d_a


def adaptive_avg_pool_rows(x, out_hw, view_hw=None, out=None):
    """README POOL=1 (README.md:68,79): every row of x [N, F], viewed as ``view_hw`` = (H, W) with H W = F (default (1, F): the 1-D pool), is
    adaptively average-pooled to ``out_hw`` = (oh, ow) -> [N, oh * ow].  C ABI: snag_adaptive_avg_pool_rows."""
    _rows(x, "x")
    N, F = x.shape
    H, W = (1, F) if view_hw is None else (int(view_hw[0]), int(view_hw[1]))
    oh, ow = (1, int(out_hw)) if isinstance(out_hw, int) else (int(out_hw[0]), int(out_hw[1]))
    if H * W != F:
        raise ValueError(f"view {H} x {W} does not cover rows of {F} features")
    if out is None:
        out = torch.empty(N, oh * ow, device=x.device, dtype=f32)
    _rows(out, "out")
    call("snag_adaptive_avg_pool_rows", ptr(x), N, x.stride(0), H, W, oh, ow, ptr(out), out.stride(0), stream())
    return out


def triple_keys(h, r, t, n_ent, n_rel):
    """Sorted int64 keys (h * n_rel + r) * n_ent + t of a triple set, for the sampler's known-triple filter."""
    k = (h.long() * n_rel + r.long()) * n_ent + t.long()
    return torch.sort(k)[0].contiguous()


def build_filter_mask(h, r, t, n_ent, n_rel, known_sorted):
    """uint8 [B, n_ent]: 1 where (h_b, r_b, x) is a known triple and x != t_b (the filtered ranking protocol).  C ABI: snag_build_filter_mask."""
    for x, nm in ((h, "h"), (r, "r"), (t, "t")):
        _chk(x, nm, dtype=torch.int32, ndim=1)
    _chk(known_sorted, "known_sorted", dtype=torch.int64, ndim=1)
    B = h.shape[0]
    mask = torch.empty(B, n_ent, device=h.device, dtype=torch.uint8)
    call("snag_build_filter_mask", ptr(h), ptr(r), ptr(t), B, int(n_ent), int(n_rel), ptr(known_sorted), known_sorted.numel(), ptr(mask), stream())
    return mask


def sample_negatives(h, r, t, n_neg, n_ent, n_rel, seed, known_sorted=None, head_or_tail=False, tick=None, out=None, distinct=False,
                     ent_list=None):
    """neg_t [B, n_neg] (and neg_h when head_or_tail) drawn on the device.  C ABI: snag_sample_negatives, or -- ``distinct=True``:
    the negatives of a positive are distinct and come from ``ent_list`` (the in-tree sampler's random.sample over the KG's own entity
    list, model/MSNEA_tools.py:59-90) -- snag_sample_negatives_distinct."""
    if distinct or ent_list is not None:
        for x, nm in ((h, "h"), (r, "r"), (t, "t")):
            _chk(x, nm, dtype=torch.int32, ndim=1)
        B = h.shape[0]
        neg_t = out if out is not None else torch.empty(B, n_neg, device=h.device, dtype=torch.int32)
        neg_h = torch.empty(B, n_neg, device=h.device, dtype=torch.int32) if head_or_tail else None
        if known_sorted is not None:
            _chk(known_sorted, "known_sorted", dtype=torch.int64, ndim=1)
        if ent_list is not None:
            _chk(ent_list, "ent_list", dtype=torch.int32, ndim=1)
        call("snag_sample_negatives_distinct", int(seed), ptr(tick), ptr(h), ptr(r), ptr(t), B, int(n_neg), int(n_ent), int(n_rel), int(head_or_tail),
             ptr(known_sorted), known_sorted.numel() if known_sorted is not None else 0, ptr(ent_list),
             ent_list.numel() if ent_list is not None else 0, ptr(neg_h), ptr(neg_t), stream())
        return (neg_h, neg_t) if head_or_tail else neg_t
    for x, nm in ((h, "h"), (r, "r"), (t, "t")):
        _chk(x, nm, dtype=torch.int32, ndim=1)
    B = h.shape[0]
    neg_t = out if out is not None else torch.empty(B, n_neg, device=h.device, dtype=torch.int32)
    neg_h = torch.empty(B, n_neg, device=h.device, dtype=torch.int32) if head_or_tail else None
    if known_sorted is not None:
        _chk(known_sorted, "known_sorted", dtype=torch.int64, ndim=1)
    call("snag_sample_negatives", int(seed), ptr(tick), ptr(h), ptr(r), ptr(t), B, int(n_neg), int(n_ent), int(n_rel), int(head_or_tail),
         ptr(known_sorted), known_sorted.numel() if known_sorted is not None else 0, ptr(neg_h), ptr(neg_t), stream())
    return (neg_h, neg_t) if head_or_tail else neg_t


# --- cross attention, the norms around a block, Muon -----------------------------------------------------------------
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # SNAG_F32, SNAG_BF16, SNAG_F16
CROSS_MAX_HEAD_DIM = 128       # SNAG_CROSS_MAX_HEAD_DIM
SANDWICH_MAX_DIM = 8192        # SNAG_SANDWICH_MAX_DIM
MUON_MAX_SIDE = 16384          # SNAG_MUON_MAX_SIDE
NORMS = {"rms": 0, "layer": 1}
_Strides = ctypes.c_int64 * 9


def _any(t, name, ndim=None):
    """A CUDA tensor of one of the three types these operators take; any strides."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in DTYPES:
        raise TypeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    if not t.is_cuda:
        raise _lib.SnagHipError(f"{name}: tensor is on {t.device}; snag_amd kernels run on the GPU only (no CPU fallback)")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name}: expected {ndim} dims, got shape {tuple(t.shape)}")
    return t


# the current stream / device as plain numbers: building torch's Stream object costs more than the launch
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


@functools.lru_cache(maxsize=None)
def _entry(name):
    return getattr(_lib.load(), name)


def _call_on(device, name, *args):
    """The entry on the current stream of the operands' device (which need not be the current one)."""
    index = device.index
    if index == _current_device():
        rc = _entry(name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = _entry(name)(*args, _raw_stream(index))
    if rc != 0:
        raise _lib.SnagHipError(f"{name} failed ({rc}): {_lib.last_error()}")


def _one_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, the first operand on {device}")


@functools.lru_cache(maxsize=4096)
def _cross_work_floats(shape, backward):
    return _lib.load().snag_cross_work_floats(*shape, backward)


def _cross_args(q, k, v, kv_lens, key_mask, scale):
    _any(q, "q", 4), _any(k, "k", 4), _any(v, "v", 4)
    (B, Lq, H, d), ks, dtype, dev = q.shape, k.shape, q.dtype, q.device
    if k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"q, k and v must share one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    if ks != v.shape or ks[0] != B or ks[3] != d:
        raise ValueError(f"k and v must be [{B}, Lk, Hkv, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    Lk, Hkv = ks[1], ks[2]
    if H == 0 or Hkv == 0 or H % Hkv:
        raise ValueError(f"{H} heads are not a multiple of {Hkv} key/value heads")
    if not 1 <= d <= CROSS_MAX_HEAD_DIM:
        raise ValueError(f"head dimension {d} is not in 1..{CROSS_MAX_HEAD_DIM}")
    if k.device != dev or v.device != dev:
        raise ValueError(f"k and v are on {k.device} and {v.device}, q on {dev}")
    qs, kt, vt = q.stride(), k.stride(), v.stride()
    if d > 1 and (qs[3] != 1 or kt[3] != 1 or vt[3] != 1):
        for t, st, name in ((q, qs, "q"), (k, kt, "k"), (v, vt, "v")):
            if st[3] != 1 and t.numel():
                raise ValueError(f"{name}: the elements of a head must be adjacent (strides {st})")
    lens_bytes = mask_ld = 0
    lens_at = mask_at = None
    if kv_lens is not None:
        _idx(kv_lens, "kv_lens", 1)
        if kv_lens.shape[0] != B:
            raise ValueError(f"kv_lens must be [{B}], got {tuple(kv_lens.shape)}")
        if kv_lens.device != dev:
            raise ValueError(f"kv_lens is on {kv_lens.device}, q on {dev}")
        lens_bytes, lens_at = kv_lens.element_size(), kv_lens.data_ptr()
    if key_mask is not None:
        if not isinstance(key_mask, torch.Tensor) or key_mask.dtype not in (torch.bool, torch.uint8):
            raise TypeError("key_mask: expected a bool (or uint8) tensor, true where a key is seen")
        if tuple(key_mask.shape) != (B, Lk):
            raise ValueError(f"key_mask must be [{B}, {Lk}], got {tuple(key_mask.shape)}")
        if not key_mask.is_cuda:
            raise _lib.SnagHipError(f"key_mask: tensor is on {key_mask.device}; snag_amd kernels run on the GPU only (no CPU fallback)")
        if key_mask.device != dev:
            raise ValueError(f"key_mask is on {key_mask.device}, q on {dev}")
        if Lk > 1 and key_mask.stride(1) != 1:
            raise ValueError("key_mask: a row's elements must be adjacent")
        mask_ld, mask_at = key_mask.stride(0) if B > 1 else Lk, key_mask.data_ptr()
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    strides = _Strides(qs[0], qs[1], qs[2], kt[0], kt[1], kt[2], vt[0], vt[1], vt[2])
    shape = (DTYPES[dtype], B, Lq, Lk, H, Hkv, d)
    return shape, (q.data_ptr(), k.data_ptr(), v.data_ptr(), *shape, ctypes.addressof(strides), lens_at, lens_bytes, mask_at, mask_ld, scale), strides


def _cross_work(shape, backward, device):
    n = _cross_work_floats(shape, int(backward))
    return (torch.empty(n, device=device, dtype=f32) if n else None), n


def cross_attention_fwd(q, k, v, kv_lens=None, key_mask=None, scale=None, want_residual=False):
    """q [B, Lq, H, d], k / v [B, Lk, Hkv, d] (any strides with adjacent head elements) -> out [B, Lq, H, d], lse [B, H, Lq] (log2), and with
    ``want_residual`` what the rounding of a 16-bit out dropped (None for fp32), for the backward.  C ABI: snag_cross_fwd."""
    shape, args, hold = _cross_args(q, k, v, kv_lens, key_mask, scale)
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    lo = torch.empty_like(out) if want_residual and q.dtype != f32 else None
    lse = torch.empty((shape[1], shape[4], shape[2]), device=q.device, dtype=f32)
    work, n = _cross_work(shape, False, q.device)
    _call_on(q.device, "snag_cross_fwd", *args, ptr(out), ptr(lo), ptr(lse), ptr(work), n)
    return (out, lse, lo) if want_residual else (out, lse)


def cross_attention_bwd(q, k, v, out, lse, d_out, kv_lens=None, key_mask=None, scale=None, out_residual=None):
    """-> d_q, d_k, d_v (dense).  C ABI: snag_cross_bwd."""
    shape, args, hold = _cross_args(q, k, v, kv_lens, key_mask, scale)
    dev, qs = q.device, q.shape
    for t, name in ((out, "out"), (d_out, "d_out"), (out_residual, "out_residual")):
        if t is None and name == "out_residual":
            continue
        _chk(t, name, dtype=q.dtype, ndim=4)
        if t.shape != qs or t.device != dev:
            raise ValueError(f"{name} must be {tuple(qs)} on {dev}, got {tuple(t.shape)} on {t.device}")
    _chk(lse, "lse", ndim=3)
    if tuple(lse.shape) != (qs[0], qs[2], qs[1]) or lse.device != dev:
        raise ValueError(f"lse must be [B, H, Lq] on {dev}, got {tuple(lse.shape)} on {lse.device}")
    dq, dk, dv = (torch.empty(t.shape, device=q.device, dtype=q.dtype) for t in (q, k, v))
    work, n = _cross_work(shape, True, q.device)
    _call_on(q.device, "snag_cross_bwd", *args, ptr(out), ptr(out_residual), ptr(lse), ptr(d_out), ptr(dq), ptr(dk), ptr(dv), ptr(work), n)
    return dq, dk, dv


@functools.lru_cache(maxsize=4096)
def _sandwich_work_floats(rows, per_gate, dim):
    return _lib.load().snag_sandwich_work_floats(rows, per_gate, dim)


def _sandwich_args(x, y, post_weight, post_bias, pre_weight, pre_bias, gate, kind):
    """-> rows, dim, (weights' dtype code), (gate dtype code), rows per gate row."""
    _any(x, "x"), _any(y, "y")
    if x.shape != y.shape or x.dim() < 1:
        raise ValueError(f"x and y must have one shape [..., dim], got {tuple(x.shape)} and {tuple(y.shape)}")
    for t, name in ((x, "x"), (y, "y")):
        if not t.is_contiguous():
            raise ValueError(f"{name}: tensor must be contiguous")
    if x.dtype not in (y.dtype, f32):
        raise TypeError(f"x (the residual stream) must be float32 or of y's type {y.dtype}, got {x.dtype}")
    if kind not in NORMS:
        raise ValueError(f"kind must be one of {sorted(NORMS)}, got {kind!r}")
    dim = x.shape[-1]
    if not 1 <= dim <= SANDWICH_MAX_DIM:
        raise ValueError(f"row width {dim} is not in 1..{SANDWICH_MAX_DIM}")
    rows = x.numel() // dim
    wt, dev = None, x.device
    if y.device != dev:
        raise ValueError(f"y is on {y.device}, x on {dev}")
    for t, name in ((post_weight, "post_weight"), (post_bias, "post_bias"), (pre_weight, "pre_weight"), (pre_bias, "pre_bias")):
        if t is None:
            continue
        _any(t, name, 1)
        if t.shape[0] != dim or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [{dim}], got {tuple(t.shape)}")
        if t.dtype not in (y.dtype, f32) or wt not in (None, t.dtype):
            raise TypeError(f"weights and biases must share one type, float32 or y's {y.dtype}; {name} is {t.dtype}")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, x on {dev}")
        wt = t.dtype
    per_gate, gt = max(rows, 1), y.dtype
    if gate is not None:
        _any(gate, "gate")
        if gate.dim() not in (1, 2) or gate.shape[-1] != dim or not gate.is_contiguous():
            raise ValueError(f"gate must be a contiguous [{dim}] or [G, {dim}], got {tuple(gate.shape)}")
        if gate.dtype not in (y.dtype, f32):
            raise TypeError(f"gate must be float32 or of y's type {y.dtype}, got {gate.dtype}")
        G = gate.shape[0] if gate.dim() == 2 else 1
        if rows and (G == 0 or rows % G):
            raise ValueError(f"{rows} rows do not divide among {G} gate rows")
        if gate.device != dev:
            raise ValueError(f"gate is on {gate.device}, x on {dev}")
        per_gate, gt = (max(rows // G, 1) if G else 1), gate.dtype
    return rows, dim, DTYPES[wt if wt is not None else y.dtype], DTYPES[gt], per_gate


def sandwich_norm_fwd(x, y, post_weight=None, pre_weight=None, post_bias=None, pre_bias=None, gate=None, res_scale=1.0, kind="rms", eps=1e-6, want_stats=True):
    """h = res_scale x + gate (post_weight N(y) + post_bias), z = pre_weight N(h) + pre_bias -> h, z, stats [rows, 4] (or None).
    C ABI: snag_sandwich_fwd."""
    plan = _sandwich_args(x, y, post_weight, post_bias, pre_weight, pre_bias, gate, kind)
    return _sandwich_fwd(plan, x, y, post_weight, pre_weight, post_bias, pre_bias, gate, res_scale, kind, eps, want_stats)


def _sandwich_fwd(plan, x, y, post_weight, pre_weight, post_bias, pre_bias, gate, res_scale, kind, eps, want_stats):
    rows, dim, wt, gt, per_gate = plan
    h, z = torch.empty_like(x), torch.empty_like(y)
    stats = torch.empty((rows, 4), device=x.device, dtype=f32) if want_stats else None
    _call_on(x.device, "snag_sandwich_fwd", ptr(x), DTYPES[x.dtype], ptr(y), DTYPES[y.dtype], rows, dim, ptr(post_weight), ptr(post_bias), ptr(pre_weight),
             ptr(pre_bias), wt, ptr(gate), gt, per_gate, float(res_scale), NORMS[kind], float(eps), ptr(h), ptr(z), ptr(stats))
    return h, z, stats


def sandwich_norm_bwd(x, y, stats, d_h, d_z, post_weight=None, pre_weight=None, post_bias=None, pre_bias=None, gate=None, res_scale=1.0, kind="rms"):
    """-> d_x, d_y, d_post_weight, d_pre_weight, d_post_bias, d_pre_bias, d_gate (None for a parameter that is None).  d_h or d_z may be None (zero).
    C ABI: snag_sandwich_bwd."""
    plan = _sandwich_args(x, y, post_weight, post_bias, pre_weight, pre_bias, gate, kind)
    for t, like, name in ((d_h, x, "d_h"), (d_z, y, "d_z")):
        if t is not None:
            _chk(t, name, dtype=like.dtype)
            if t.shape != like.shape:
                raise ValueError(f"{name} must be {tuple(like.shape)}, got {tuple(t.shape)}")
    _chk(stats, "stats", ndim=2)
    if tuple(stats.shape) != (plan[0], 4):
        raise ValueError(f"stats must be [{plan[0]}, 4], got {tuple(stats.shape)}")
    _one_device(x.device, stats=stats, d_h=d_h, d_z=d_z)
    return _sandwich_bwd(plan, x, y, stats, d_h, d_z, post_weight, pre_weight, post_bias, pre_bias, gate, res_scale, kind)


def _sandwich_bwd(plan, x, y, stats, d_h, d_z, post_weight, pre_weight, post_bias, pre_bias, gate, res_scale, kind):
    rows, dim, wt, gt, per_gate = plan
    new = torch.empty_like if rows else torch.zeros_like
    dx, dy, dpw, dqw, dpb, dqb, dg = (None if t is None else new(t) for t in (x, y, post_weight, pre_weight, post_bias, pre_bias, gate))
    n = _sandwich_work_floats(rows, per_gate, dim)
    work = torch.empty(n, device=x.device, dtype=f32)
    _call_on(x.device, "snag_sandwich_bwd", ptr(x), DTYPES[x.dtype], ptr(y), DTYPES[y.dtype], rows, dim, ptr(post_weight), ptr(post_bias), ptr(pre_weight), wt,
             ptr(gate), gt, per_gate, float(res_scale), NORMS[kind], ptr(stats), ptr(d_h), ptr(d_z), ptr(dx), ptr(dy), ptr(dpw), ptr(dpb), ptr(dqw), ptr(dqb),
             ptr(dg), ptr(work), n)
    return dx, dy, dpw, dqw, dpb, dqb, dg


def _matrices(ts, name, dtype=None, shapes=None, device=None):
    """A list of contiguous 2-D CUDA tensors of one type on one device -> (list, shapes)."""
    ts = list(ts)
    if ts:
        dtype, device = dtype or _any(ts[0], f"{name}[0]").dtype, device or ts[0].device
    got = []
    for i, t in enumerate(ts):
        _any(t, name, 2)
        s = t.shape
        if t.dtype != dtype:
            raise TypeError(f"{name}[{i}]: expected {dtype}, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name}[{i}]: tensor must be contiguous")
        if shapes is not None and s != shapes[i]:
            raise ValueError(f"{name}[{i}] must be {tuple(shapes[i])}, got {tuple(s)}")
        if not (1 <= s[0] <= MUON_MAX_SIDE and 1 <= s[1] <= MUON_MAX_SIDE):
            raise ValueError(f"{name}[{i}]: sides must be in 1..{MUON_MAX_SIDE}, got {tuple(s)}")
        if t.device != device:
            raise ValueError(f"{name}[{i}] is on {t.device}, the first matrix on {device}")
        got.append(s)
    return ts, got


def _disjoint(written, read):
    """Nothing that is written shares memory with anything else in the call."""
    spans = sorted([(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), True) for t in written] +
                   [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), False) for t in read])
    any_end = written_end = 0
    for start, end, writes in spans:
        if start < written_end or (writes and start < any_end):
            raise ValueError("a matrix is listed twice, or shares memory with another one of the call")
        any_end = max(any_end, end)
        if writes:
            written_end = max(written_end, end)


def _muon_lists(*lists):
    return [(ctypes.c_void_p * len(ts))(*[t.data_ptr() for t in ts]) for ts in lists]


@functools.lru_cache(maxsize=256)
def _muon_shapes(shapes):
    """Host arrays of the shapes and the workspace they need (by shape alone)."""
    n = len(shapes)
    rows, cols = (ctypes.c_int32 * n)(*[s[0] for s in shapes]), (ctypes.c_int32 * n)(*[s[1] for s in shapes])
    return rows, cols, _lib.load().snag_muon_work_bytes(ctypes.addressof(rows), ctypes.addressof(cols), n)


def orthogonalize(gs, outs=None, steps=5, eps=1e-7):
    """Newton-Schulz orthogonalisation of a list of matrices of one type -> list (or into ``outs``; outs[i] may be gs[i]).
    C ABI: snag_orthogonalize."""
    gs, shapes = _matrices(gs, "gs")
    if not 1 <= int(steps) <= 100:
        raise ValueError(f"steps must be in 1..100, got {steps}")
    if outs is None:
        outs = [torch.empty_like(g) for g in gs]
    else:
        outs = list(outs)
        if len(outs) != len(gs):
            raise ValueError(f"{len(gs)} matrices, {len(outs)} outputs")
        if gs:
            _matrices(outs, "outs", gs[0].dtype, shapes, gs[0].device)
            _disjoint(outs, [g for g, o in zip(gs, outs) if g.data_ptr() != o.data_ptr()])
            torch.autograd.graph.increment_version(outs)
    if not gs:
        return outs
    rows, cols, n = _muon_shapes(tuple(shapes))
    work = torch.empty(n, device=gs[0].device, dtype=torch.uint8)
    pg, po = _muon_lists(gs, outs)
    _call_on(gs[0].device, "snag_orthogonalize", ctypes.addressof(pg), ctypes.addressof(po), ctypes.addressof(rows), ctypes.addressof(cols), len(gs),
             DTYPES[gs[0].dtype], int(steps), float(eps), ptr(work), n)
    return outs


def muon_step(weights, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, match_rms=False, steps=5, eps=1e-7):
    """One Muon update, in place on ``weights`` (one type) and ``momenta`` (fp32); ``grads`` have the weights' type.  C ABI: snag_muon_step."""
    weights, shapes = _matrices(weights, "weights")
    grads, momenta = list(grads), list(momenta)
    if len(grads) != len(weights) or len(momenta) != len(weights):
        raise ValueError(f"{len(weights)} weights, {len(grads)} gradients, {len(momenta)} momenta")
    if not 1 <= int(steps) <= 100:
        raise ValueError(f"steps must be in 1..100, got {steps}")
    if not 0.0 <= momentum < 1.0:
        raise ValueError(f"momentum must be in [0, 1), got {momentum}")
    if not weights:
        return
    dev = weights[0].device
    _matrices(grads, "grads", weights[0].dtype, shapes, dev), _matrices(momenta, "momenta", f32, shapes, dev)
    _disjoint(weights + momenta, grads)
    torch.autograd.graph.increment_version(weights + momenta)      # a graph that saved one of them must not run on the new values
    rows, cols, n = _muon_shapes(tuple(shapes))
    work = torch.empty(n, device=dev, dtype=torch.uint8)
    pw, pg, pm = _muon_lists(weights, grads, momenta)
    _call_on(weights[0].device, "snag_muon_step", ctypes.addressof(pw), ctypes.addressof(pg), ctypes.addressof(pm), ctypes.addressof(rows), ctypes.addressof(cols),
             len(weights), DTYPES[weights[0].dtype], float(lr), float(momentum), int(nesterov), float(weight_decay), int(match_rms), int(steps), float(eps),
             ptr(work), n)
