"""A cross-attention block: tokens read an encoder's states of another length.

The reference fuses one vector per modality (model/SNAG_tools.py:23-51: at most six tokens an entity, attended by themselves).  Here an
entity's tokens read ANY number of states per modality -- image patches, words, attribute values -- with the block's norms, gate and
residual fused around it.  All arithmetic is in the HIP library, forward and backward; fp32, bf16 and fp16; there is no CPU path.

  cross_attention(q, k, v, ...)   attention of queries over keys and values of another length
  sandwich_norm(x, y, ...)        the norm after a block, its gate, the residual and the next block's norm, in one pass
  CrossModalLayer                 the two with fp32 projections and a feed-forward block: one layer of a deeper fusion
"""
import functools
import math

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .projection import Linear, ProjectionHead

LN2 = math.log(2.0)


def _note_stream(out):
    """A gradient node belongs to the stream it was made on, a leaf's to that of the first live graph that reaches it.  A backward captured on
    another stream would pull that stream into the capture, and torch then ends the process.  torch does not tell a node's stream, so each call
    leaves its own on the nodes it reads from, and a call inside a capture looks through the whole graph below it: one that reaches a node left by
    an eager call on another stream is refused.  Graphs that other operations alone built of the same leaves are not seen."""
    st, capturing = ops._raw_stream(out.device.index), torch.cuda.is_current_stream_capturing()
    below = [node for node, _ in out.grad_fn.next_functions if node is not None]
    for node in below:
        node.metadata.setdefault("snag_stream", st)
    if not capturing:
        return
    seen = set(below)
    while below:
        node = below.pop()
        if node.metadata.get("snag_stream", st) != st:
            raise _lib.SnagHipError("a backward cannot be captured while an eager graph of the same leaves lives on another stream: drop that graph's outputs first")
        for n, _ in node.next_functions:
            if n is not None and n not in seen:
                seen.add(n)
                below.append(n)


def _noted(out):
    """A projection's output, its leaves' nodes noted as those of the operators beside it."""
    if out.grad_fn is not None:
        _note_stream(out)
    return out


def _first_order(backward):
    """once_differentiable without its bookkeeping where no graph of the backward is asked for."""
    recorded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


def _no_tangents(name, *ts):
    """Forward-mode derivatives have no formula here, and a call past the autograd function would drop them without a word."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise _lib.SnagHipError(f"{name}: forward-mode derivatives are not implemented")


class _CrossAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kv_lens, key_mask, scale, want_lse):
        out, lse, lo = ops.cross_attention_fwd(q, k, v, kv_lens, key_mask, scale, want_residual=True)
        ctx.save_for_backward(q, k, v, kv_lens, key_mask, out, lse, lo)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        if not want_lse:
            return out
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @_first_order
    def backward(ctx, d_out, *_):
        if d_out is None:
            return (None,) * 7
        q, k, v, kv_lens, key_mask, out, lse, lo = ctx.saved_tensors
        dq, dk, dv = ops.cross_attention_bwd(q, k, v, out, lse, d_out.contiguous(), kv_lens, key_mask, ctx.scale, lo)
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None, None


def cross_attention(q, k, v, kv_lens=None, key_mask=None, scale=None, return_lse=False):
    """Attention of q [B, Lq, H, d] over k, v [B, Lk, Hkv, d] -> [B, Lq, H, d], differentiable (backward, once) in q, k and v.

    H is a multiple of Hkv (query head h reads key/value head h // (H / Hkv)), d <= 128.  Any strides whose last one is 1; fp32, bf16 or fp16.
    ``kv_lens`` [B] (int32 / int64, on the device): keys at and behind it are not seen; ``key_mask`` [B, Lk] (bool): nor are those that are
    False.  Unseen keys may hold anything.  A query that sees no key gets zeros, and gives none of its gradient on.  ``scale`` defaults to d ** -0.5.
    Scores, softmax statistics and sums are fp32; with more than a few rows per key/value head, 16-bit inputs round the probabilities (and in the
    backward d scores) to their type for the second product: bf16 gradients are 2.4e-3 off the 64-bit ones, their own rounding alone 1.7e-3.
    ``return_lse`` adds the natural log-sum-exp of every row's scores [B, H, Lq] (-inf where no key is seen), not differentiable."""
    if forward_ad._current_level >= 0:
        _no_tangents("cross_attention", q, k, v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        got = _CrossAttentionFn.apply(q, k, v, kv_lens, key_mask, scale, return_lse)
        out = got[0] if return_lse else got
        _note_stream(out)
    else:
        got = ops.cross_attention_fwd(q, k, v, kv_lens, key_mask, scale)
        out = got[0]
    return (out, got[1] * LN2) if return_lse else out


class _SandwichNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, post_weight, pre_weight, post_bias, pre_bias, gate, res_scale, kind, eps):
        plan = ops._sandwich_args(x, y, post_weight, post_bias, pre_weight, pre_bias, gate, kind)
        h, z, stats = ops._sandwich_fwd(plan, x, y, post_weight, pre_weight, post_bias, pre_bias, gate, res_scale, kind, eps, True)
        ctx.save_for_backward(x, y, stats, post_weight, pre_weight, post_bias, pre_bias, gate)
        ctx.cfg = (plan, res_scale, kind)
        ctx.set_materialize_grads(False)
        return h, z

    @staticmethod
    @_first_order
    def backward(ctx, d_h, d_z):
        x, y, stats, post_weight, pre_weight, post_bias, pre_bias, gate = ctx.saved_tensors
        plan, res_scale, kind = ctx.cfg
        grads = ops._sandwich_bwd(plan, x, y, stats, None if d_h is None else d_h.contiguous(), None if d_z is None else d_z.contiguous(),
                                  post_weight, pre_weight, post_bias, pre_bias, gate, res_scale, kind)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None)


def _wants_grad(*ts):
    return any(t is not None and t.requires_grad for t in ts)


def sandwich_norm(x, y, post_weight=None, pre_weight=None, post_bias=None, pre_bias=None, gate=None, res_scale=1.0, kind="rms", eps=1e-6):
    """The norms around a block: h = res_scale x + gate (post_weight N(y) + post_bias), z = pre_weight N(h) + pre_bias -> (h, z).

    x: the residual stream, y: the block's output, [..., dim] (dim <= 8192); h continues the stream, z enters the next block.  ``kind`` "rms"
    (v / sqrt(mean v^2 + eps)) or "layer" (around the mean, biased variance).  ``gate`` [dim], or [G, dim] whose rows serve rows / G
    neighbouring rows each (one gate per sequence, or per row).  x may stay fp32 while y is 16-bit; h has x's type, z y's.  Weights and biases
    share one type, fp32 or y's; so does the gate.  Differentiable (backward, once) in every tensor."""
    if forward_ad._current_level >= 0:
        _no_tangents("sandwich_norm", x, y, post_weight, pre_weight, post_bias, pre_bias, gate)
    if not (x.is_contiguous() and y.is_contiguous()):
        x, y = x.contiguous(), y.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or y.requires_grad or _wants_grad(post_weight, pre_weight, post_bias, pre_bias, gate)):
        h, z = _SandwichNormFn.apply(x, y, post_weight, pre_weight, post_bias, pre_bias, gate, res_scale, kind, eps)
        _note_stream(h)
        return h, z
    return ops.sandwich_norm_fwd(x, y, post_weight, pre_weight, post_bias, pre_bias, gate, res_scale, kind, eps, want_stats=False)[:2]


class _SandwichNorm(nn.Module):
    """Parameters of one sandwich_norm: both norms' weights and the gate (one per channel, small at the start: the layer begins near the identity)."""

    def __init__(self, dim, gate, res_scale, kind, eps):
        super().__init__()
        self.post_weight = nn.Parameter(torch.ones(dim))
        self.pre_weight = nn.Parameter(torch.ones(dim))
        self.gate = nn.Parameter(torch.full((dim,), float(gate)))
        self.res_scale, self.kind, self.eps = float(res_scale), kind, float(eps)

    def forward(self, x, y):
        return sandwich_norm(x, y, self.post_weight, self.pre_weight, gate=self.gate, res_scale=self.res_scale, kind=self.kind, eps=self.eps)


class CrossModalLayer(nn.Module):
    """One layer in which the tokens of an entity read a modality's states: cross attention, then a feed-forward block, each inside a
    sandwich norm.  fp32, like the modules beside it (``MformerFusion`` reads the M vectors this layer puts out).

    ``layer(x, states, kv_lens, key_mask) -> (h, z)``: x [N, M, D] tokens, states [N, L, state_dim]; h is the residual stream, z its norm,
    which the next layer takes as ``z`` (the first layer's tokens are taken as they are)."""

    def __init__(self, dim, num_heads, state_dim=None, kv_heads=None, intermediate_size=None, gate=0.1, res_scale=1.0, kind="rms", eps=1e-6):
        super().__init__()
        kv_heads = num_heads if kv_heads is None else kv_heads
        if dim % num_heads or num_heads % kv_heads:
            raise ValueError(f"hidden size {dim} is not a multiple of {num_heads} heads, or those not of {kv_heads} key/value heads")
        state_dim, head = dim if state_dim is None else state_dim, dim // num_heads
        if head > ops.CROSS_MAX_HEAD_DIM:
            raise ValueError(f"head dimension {head} > {ops.CROSS_MAX_HEAD_DIM}")
        self.num_heads, self.kv_heads, self.head = num_heads, kv_heads, head
        self.query = Linear(dim, dim)
        self.key = Linear(state_dim, kv_heads * head)
        self.value = Linear(state_dim, kv_heads * head)
        self.output = Linear(dim, dim)
        self.attention_norm = _SandwichNorm(dim, gate, res_scale, kind, eps)
        self.feed_forward = ProjectionHead(dim, 4 * dim if intermediate_size is None else intermediate_size, dim, 0.0)
        self.feed_forward_norm = _SandwichNorm(dim, gate, res_scale, kind, eps)

    def forward(self, x, states, kv_lens=None, key_mask=None, z=None):
        N, M, D = x.shape
        L = states.shape[1]
        z = x if z is None else z
        flat = lambda t: t.reshape(-1, t.shape[-1])
        q = _noted(self.query(flat(z))).view(N, M, self.num_heads, self.head)
        k = _noted(self.key(flat(states))).view(N, L, self.kv_heads, self.head)
        v = _noted(self.value(flat(states))).view(N, L, self.kv_heads, self.head)
        a = cross_attention(q, k, v, kv_lens, key_mask)
        x, z = self.attention_norm(x, _noted(self.output(a.reshape(N * M, D))).view(N, M, D))
        f = _noted(self.feed_forward(flat(z)))
        return self.feed_forward_norm(x, f.view(N, M, D))
