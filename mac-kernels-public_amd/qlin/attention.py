"""The attention side of a block, between its packed QKV projection and its output projection.

  rope_frequencies      the pairs' frequencies and axes of a rotation (made once for a model)
  axis_rope             rotation of q and k by positions on one or several axes (text; time, height, width)
  qk_norm_rope          per-head RMS norms of q and k with the rotation in the same pass; _grad its backward,
                        _store the form that writes k and v straight into a paged cache
  paged_plan            pages, slots and positions of a step over the cache, from request lengths on the GPU
  paged_attention       attention of one new token a row over the cache

q, k and v are [.., heads, D] in fp16, bf16 or fp32 (attention: fp16, bf16); the slices of a fused projection's
output go in as they are.  A cache is [blocks, page, kv heads, D] in any memory order that keeps D's values together
(allocate [blocks, kv heads, page, D] and transpose(1, 2) to keep a head's page in one piece).  Every op runs on the
current stream and returns new tensors, except that caches and block tables are written in place.  Calls that
the kernels do not take raise NoCapableBackendError, malformed ones ValueError, as the linears do.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib, ops
from .exceptions import NoCapableBackendError
from .ops import _check_device, _disabled, _fast_error


class PagedPlan(NamedTuple):
    """What paged_plan fills.  N places for the step's new tokens, B requests."""
    slots: torch.Tensor      # int64 [N]: block * page + place in it, -1 for none
    positions: torch.Tensor  # int32 [N]: the token's position in its request
    rows: torch.Tensor       # int32 [N]: its request
    starts: torch.Tensor     # int32 [B + 1]: where each request's tokens start among the N
    lengths: torch.Tensor    # int32 [B]: tokens of each request after the step
    used: torch.Tensor       # int32 [1]: pages taken from the free list (more than it holds: it was too short)


def rope_frequencies(sizes, theta=10000.0, *, shared=False, device=None):
    """(inv_freq float32 [P], axis int32 [P]) for a rotation of `sizes` values on each axis (P = sum(sizes) / 2).
    Each axis has its own ladder theta^(-2j / size), or with `shared` its section of one ladder over all sizes (the
    form of language models that see images)."""
    sizes = [int(n) for n in ((sizes,) if isinstance(sizes, int) else sizes)]
    if not sizes or any(n < 0 or n % 2 for n in sizes):
        raise ValueError(f"rope_frequencies: sizes {sizes} are not even numbers of values")
    if shared:
        total = sum(sizes)
        exponent = torch.arange(0, total, 2, dtype=torch.float64) / max(total, 1)
    else:
        exponent = torch.cat([torch.arange(0, n, 2, dtype=torch.float64) / max(n, 1) for n in sizes])
    axis = torch.cat([torch.full((n // 2,), i, dtype=torch.int32) for i, n in enumerate(sizes)])
    return (float(theta) ** -exponent).to(torch.float32).to(device), axis.to(device)


def _dense(t):
    """t with unit stride along its last dimension (a copy if need be)."""
    return t if t.dim() == 0 or t.size(-1) <= 1 or t.stride(-1) == 1 else t.contiguous()


def _heads(op, t, name):
    """[.., heads, D] as [tokens, heads, D]."""
    if t.dim() < 3:
        raise ValueError(f"{op}: {name} must be [.., heads, D], it has {t.dim()} dimensions")
    return _dense(t if t.dim() == 3 else t.reshape(math.prod(t.shape[:-2]), *t.shape[-2:]))  # -1 has no meaning without values


def _vector(t, dtype=None):
    if t is None:
        return None
    t = t if dtype is None or t.dtype == dtype else t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def _desc(op, t):
    if t is not None and t.dtype not in _lib._TORCH_DT:
        raise NoCapableBackendError(op, {"hip": f"dtype {t.dtype} unsupported"})
    return _lib.desc(t)


def _flags(interleaved, inverse=False):
    return (_lib.ROPE_INTERLEAVED if interleaved else 0) | (_lib.ROPE_INVERSE if inverse else 0)


def _run(op, name, device, *args):
    """The C ABI entry point `name`; tensors (and None) become descriptors, valid for this call."""
    args = [a if isinstance(a, (int, float)) else _desc(op, a) for a in args]
    _lib.check(getattr(_lib.load(), name)(*args, _lib.stream_of(device)), op)


def axis_rope(q, k, positions, inv_freq, axis=None, *, interleaved=False, inverse=False):
    """(rotated q, rotated k) in fp32 with one rounding; k may be None.  Pair i turns by positions[axis[i], t] *
    inv_freq[i] (positions int32, int64 or float32 [axes, tokens] or [tokens]; axis None: the first), `inverse` by its
    negative.  Pairs are (i, i + P), or (2i, 2i + 1) when `interleaved`; the values from 2P on pass through."""
    op = "axis_rope"
    _disabled(op)
    if ops._FAST is not None:
        try:
            return ops._FAST.axis_rope(q, k, positions, inv_freq, axis, _flags(interleaved, inverse))
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, q, k, positions, inv_freq, axis)
    q3, k3 = _heads(op, q, "q"), None if k is None else _heads(op, k, "k")
    qo = torch.empty(q3.shape, dtype=q.dtype, device=q.device)
    ko = None if k is None else torch.empty(k3.shape, dtype=k.dtype, device=q.device)
    _run(op, "qlin_axis_rope", q.device, q3, k3, positions, _vector(inv_freq, torch.float32), _vector(axis, torch.int32),
         _flags(interleaved, inverse), qo, ko)
    return qo.view(q.shape), None if k is None else ko.view(k.shape)


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, axis=None, *, eps=1e-6, interleaved=False):
    """(rotate(q_weight * q / rms(q)), the same of k), rms(x) = sqrt(mean(x^2) + eps) over each head, in fp32 with one
    rounding.  Weights [D] or None (1); k may be None.  The rotation's arguments are those of axis_rope."""
    op = "qk_norm_rope"
    _disabled(op)
    if ops._FAST is not None:
        try:
            return ops._FAST.qk_norm_rope(q, k, q_weight, k_weight, float(eps), positions, inv_freq, axis, _flags(interleaved))
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, q, k, q_weight, k_weight, positions, inv_freq, axis)
    q3, k3 = _heads(op, q, "q"), None if k is None else _heads(op, k, "k")
    qo = torch.empty(q3.shape, dtype=q.dtype, device=q.device)
    ko = None if k is None else torch.empty(k3.shape, dtype=k.dtype, device=q.device)
    _run(op, "qlin_qk_norm_rope", q.device, q3, k3, _vector(q_weight), _vector(k_weight), float(eps), positions,
         _vector(inv_freq, torch.float32), _vector(axis, torch.int32), _flags(interleaved), qo, ko)
    return qo.view(q.shape), None if k is None else ko.view(k.shape)


def qk_norm_rope_store(q, k, v, q_weight, k_weight, positions, inv_freq, slots, k_cache, v_cache, axis=None, *, eps=1e-6,
                       interleaved=False):
    """qk_norm_rope with k and v written into the caches [blocks, page, kv heads, D] at `slots` (int64 or int32 [tokens],
    paged_plan's; below 0 or past the cache: not stored).  Returns the rotated q.  eps None: no norms, the
    rotation alone (the weights must be None)."""
    op = "qk_norm_rope_store"
    _disabled(op)
    e = -1.0 if eps is None else float(eps)
    if eps is not None and not e >= 0.0:
        raise ValueError(f"{op}: eps must not be negative")
    if ops._FAST is not None:
        try:
            return ops._FAST.qk_norm_rope_store(q, k, v, q_weight, k_weight, e, positions, inv_freq, axis, _flags(interleaved),
                                                slots, k_cache, v_cache)
        except ops._FastError as err:
            raise _fast_error(op, err) from None
    _check_device(op, q, k, v, q_weight, k_weight, positions, inv_freq, axis, slots, k_cache, v_cache)
    q3 = _heads(op, q, "q")
    qo = torch.empty(q3.shape, dtype=q.dtype, device=q.device)
    _run(op, "qlin_qk_norm_rope_store", q.device, q3, _heads(op, k, "k"), _heads(op, v, "v"), _vector(q_weight),
         _vector(k_weight), e, positions, _vector(inv_freq, torch.float32), _vector(axis, torch.int32), _flags(interleaved),
         slots, qo, k_cache, v_cache)
    return qo.view(q.shape)


def qk_norm_rope_grad(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, axis=None, *, eps=1e-6,
                      interleaved=False, weight_grads=True):
    """(dq, dk, dq_weight, dk_weight) of qk_norm_rope from the gradients of its outputs.  The weights' gradients are summed
    in fp32 in a fixed order and rounded to the weight's dtype; None where there is no weight, and with `weight_grads`
    False (frozen norms; a pair says it for q's and k's apart)."""
    op = "qk_norm_rope_grad"
    _disabled(op)
    of_q, of_k = weight_grads if isinstance(weight_grads, (tuple, list)) else (weight_grads, weight_grads)
    if ops._FAST is not None:
        try:
            return ops._FAST.qk_norm_rope_grad(dq_out, dk_out, q, k, q_weight, k_weight, float(eps), positions, inv_freq, axis,
                                               _flags(interleaved), bool(of_q), bool(of_k))
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, axis)
    q3, k3 = _heads(op, q, "q"), None if k is None else _heads(op, k, "k")
    dq = torch.empty(q3.shape, dtype=q.dtype, device=q.device)
    dk = None if k is None else torch.empty(k3.shape, dtype=k.dtype, device=q.device)
    wq, wk = _vector(q_weight), _vector(k_weight)
    dwq = torch.empty_like(wq) if of_q and wq is not None else None
    dwk = torch.empty_like(wk) if of_k and wk is not None else None
    ws = None
    if dwq is not None or dwk is not None:
        ws = ops._workspace(_lib.OP_QK_NORM_ROPE_GRAD, q3.shape[0], q3.shape[1] + (0 if k is None else k3.shape[1]),
                            q3.shape[2], 0, q3)
    dt = torch.float32
    gq, gk = _heads(op, dq_out, "dq_out"), None if dk_out is None else _heads(op, dk_out, "dk_out")
    _run(op, "qlin_qk_norm_rope_grad", q.device, gq, gk, q3, k3, wq, wk, float(eps), positions, _vector(inv_freq, dt),
         _vector(axis, torch.int32), _flags(interleaved), dq, dk, dwq, dwk, ws.data_ptr() if ws is not None else 0,
         ws.numel() if ws is not None else 0)
    return dq.view(q.shape), None if k is None else dk.view(k.shape), dwq, dwk


def paged_plan(context, added, block_table, free_blocks, page, tokens):
    """The tables of a step: request b has context[b] tokens in the cache and gets added[b] (int32 [B], on the GPU).  Pages
    that the requests lack are taken from free_blocks (int32 [F]) in the order of the requests and written into block_table
    (int32 [B, W], in place).  `tokens`: the places to fill, at least the new tokens' number (more, as for a captured
    graph of a fixed size: the rest gets -1).  Returns a PagedPlan."""
    op = "paged_plan"
    _disabled(op)
    if ops._FAST is not None:
        try:
            return PagedPlan._make(ops._FAST.paged_plan(context, added, block_table, free_blocks, int(page), int(tokens)))
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, context, added, block_table, free_blocks)
    if int(tokens) < 0:
        raise ValueError(f"{op}: tokens must not be negative")
    dev, n = context.device, int(tokens)
    b = context.shape[0] if context.dim() == 1 else 0
    i32 = dict(dtype=torch.int32, device=dev)
    p = PagedPlan(torch.empty(n, dtype=torch.int64, device=dev), torch.empty(n, **i32), torch.empty(n, **i32),
                  torch.empty(b + 1, **i32), torch.empty(b, **i32), torch.empty(1, **i32))
    _run(op, "qlin_paged_plan", dev, context, added, free_blocks, int(page), block_table, p.slots, p.positions, p.rows, p.starts,
         p.lengths, p.used)
    return p


def paged_attention(q, k_cache, v_cache, block_table, lengths, *, scale=None, window=0, out=None):
    """softmax(scale * q k^T) v of one new token a row: q [rows, heads, D], the first lengths[b] tokens of row b's pages (the
    last `window` of them when window > 0).  block_table int32 [rows, W] (expanded rows are fine: a prompt's tokens share
    one, with lengths 1, 2, ...), lengths int32 [rows].  scale None: D ** -0.5.  `out`: where to write, shaped
    like q.  A row without a token gives zeros."""
    op = "paged_attention"
    _disabled(op)
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0  # no head size: refused below
    scale = float(scale)
    if ops._FAST is not None:
        try:
            return ops._FAST.paged_attention(q, k_cache, v_cache, block_table, lengths, scale, int(window), out)
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, q, k_cache, v_cache, block_table, lengths, out)
    if q.dim() != 3 or k_cache.dim() != 4:
        raise ValueError(f"{op}: q must be [rows, heads, D] and the caches [blocks, page, kv heads, D]")
    q3 = _dense(q)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ws = ops._workspace(_lib.OP_PAGED_ATTENTION, q.shape[0], q.shape[1], q.shape[2], k_cache.shape[2], q3)
    _run(op, "qlin_paged_attention", q.device, q3, k_cache, v_cache, block_table, lengths, scale, int(window), out,
         ws.data_ptr(), ws.numel())
    return out


# ------------------------------------------------------------------------------------------------
# Training
# ------------------------------------------------------------------------------------------------

class _AxisRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, axis, interleaved, inverse):
        ctx.save_for_backward(positions, inv_freq, axis)
        ctx.conf = (bool(interleaved), bool(inverse))
        return axis_rope(q, k, positions, inv_freq, axis, interleaved=interleaved, inverse=inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        interleaved, inverse = ctx.conf
        # itself a rotation with gradients: a second derivative goes on through it
        dq, dk = _AxisRope.apply(gq, gk, *ctx.saved_tensors, interleaved, not inverse)
        return dq, dk, None, None, None, None, None


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, inv_freq, axis, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, inv_freq, axis)
        ctx.conf = (float(eps), bool(interleaved))
        return qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, axis, eps=eps, interleaved=interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, positions, inv_freq, axis = ctx.saved_tensors
        eps, interleaved = ctx.conf
        need = ctx.needs_input_grad
        dq, dk, dwq, dwk = qk_norm_rope_grad(gq, gk, q, k, q_weight, k_weight, positions, inv_freq, axis, eps=eps,
                                             interleaved=interleaved, weight_grads=(need[2], need[3]))
        return (dq if need[0] else None, dk if need[1] else None, dwq if need[2] else None, dwk if need[3] else None,
                None, None, None, None, None)


def axis_rope_trainable(q, k, positions, inv_freq, axis=None, interleaved=False):
    """axis_rope with gradients for q and k, of any order."""
    return _AxisRope.apply(q, k, positions, inv_freq, axis, interleaved, False)


def qk_norm_rope_trainable(q, k, q_weight, k_weight, positions, inv_freq, axis=None, eps=1e-6, interleaved=False):
    """qk_norm_rope with gradients for q, k and the weights (a frozen weight's is not formed); first derivatives
    only."""
    return _QkNormRope.apply(q, k, q_weight, k_weight, positions, inv_freq, axis, eps, interleaved)
