"""The MLP side of a block: what stands before, between and beside its packed linears.

  add_rms_norm          root-mean-square norm of a row with the residual's addition; _int8 with an output in 8 bits for a
                        linear over int8 rows, _grad its backward
  gated_act             gated activation (SiLU, GELU in its tanh form); _int8 and _grad as above
  w8a8_int8_linear      product of int8 rows with scales for each token and channel

Rows are [.., values] in fp16, bf16 or fp32; the halves of a fused projection's output go in as they are.  The 8-bit outputs
are (codes int8 [.., values], scale fp32 [.., 1]): codes * scale stands for the row, which goes through the ConvRot rotation
first where the linear's weights are stored rotated.  Every op runs on the current stream and returns new tensors.
Calls that the kernels do not take raise NoCapableBackendError, malformed ones ValueError, as the linears do.
"""
from __future__ import annotations

import math

import torch

from . import _lib, ops
from .attention import _desc, _run, _vector
from .autograd import int8_linear_grad_input
from .exceptions import NoCapableBackendError
from .ops import _check_device, _disabled, _fast_error, _residual_args, quantize_int8_rowwise

ACTIVATIONS = {"silu": 0, "gelu_tanh": 1}


def _act(op, act):
    try:
        return ACTIVATIONS[act]
    except (KeyError, TypeError):
        raise NoCapableBackendError(op, {"hip": f"activation {act!r} unsupported ({', '.join(ACTIVATIONS)})"}) from None


def _rows(op, t, name, shape=None):
    """[.., values] as [rows, values] with unit stride along a row (a copy if need be)."""
    if t is None:
        return None
    if t.dim() < 1:
        raise ValueError(f"{op}: {name} must be [.., values]")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{op}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    t = t if t.dim() == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])  # -1 has no meaning without values
    return t if t.size(1) <= 1 or t.stride(1) == 1 else t.contiguous()


def _dtype(op, t, name, *known):
    """Declines t before its dtype is looked up for a workspace's size."""
    if t.dtype not in known:
        raise NoCapableBackendError(op, {"hip": f"{name} dtype {t.dtype} unsupported"})


def _codes(shape, device):
    q = torch.empty(shape, dtype=torch.int8, device=device)
    return q, torch.empty((*shape[:-1], 1), dtype=torch.float32, device=device)


def _flat(t):
    return None if t is None else t.view(math.prod(t.shape[:-1]), t.shape[-1])


def add_rms_norm(x, residual=None, weight=None, *, eps=1e-6):
    """(y, h): h = x + residual, y = weight * h / sqrt(mean(h^2) + eps) over the last dimension, in fp32 with one rounding each
    (the norm is that of the unrounded sum).  residual in x's dtype or fp32, which is h's; without one h is x.  weight
    [values] or None (1)."""
    op = "add_rms_norm"
    _disabled(op)
    if ops._FAST is not None:
        try:
            return ops._FAST.add_rms_norm(x, residual, weight, float(eps))
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, x, residual, weight)
    x2, r2 = _rows(op, x, "x"), _rows(op, residual, "residual", x.shape)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = x if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    _run(op, "qlin_add_rms_norm", x.device, x2, r2, _vector(weight), float(eps), _flat(y), None if residual is None else _flat(h))
    return y, h


def add_rms_norm_int8(x, residual=None, weight=None, *, eps=1e-6, convrot_groupsize=0):
    """(codes, scale, h): add_rms_norm with y in 8 bits."""
    op = "add_rms_norm_int8"
    _disabled(op)
    if ops._FAST is not None:
        try:
            return ops._FAST.add_rms_norm_int8(x, residual, weight, float(eps), int(convrot_groupsize))
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, x, residual, weight)
    x2, r2 = _rows(op, x, "x"), _rows(op, residual, "residual", x.shape)
    q, scale = _codes(x.shape, x.device)
    h = x if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    _run(op, "qlin_add_rms_norm_int8", x.device, x2, r2, _vector(weight), float(eps), int(convrot_groupsize), _flat(q), _flat(scale),
         None if residual is None else _flat(h))
    return q, scale, h


def add_rms_norm_grad(dy, dh, h, weight=None, *, eps=1e-6, weight_grad=True):
    """(dx, dweight) of add_rms_norm from the gradients of y and of h (dh None: none reaches h), h as the forward call gave
    it.  dx is x's and the residual's gradient both, in h's dtype.  dweight is summed in fp32 in a fixed order and rounded to the
    weight's dtype; None where there is no weight, and with `weight_grad` False (a frozen norm).

    h is taken as it was stored, where the forward norm is that of the unrounded sum.  In 16 bits its rounding makes dweight about 1.5
    times as far from the gradient through the sum as rounding it to 16 bits alone does (dx hardly, unless dy lies along h); a
    residual in fp32 avoids it."""
    op = "add_rms_norm_grad"
    _disabled(op)
    if ops._FAST is not None:
        try:
            return ops._FAST.add_rms_norm_grad(dy, dh, h, weight, float(eps), bool(weight_grad))
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, dy, dh, h, weight)
    _dtype(op, dy, "dy", *ops._FLOAT)
    g2, d2, h2 = _rows(op, dy, "dy"), _rows(op, dh, "dh", dy.shape), _rows(op, h, "h", dy.shape)
    dx = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    w = _vector(weight)
    dw = torch.empty_like(w) if weight_grad and w is not None else None
    ws = None if dw is None else ops._workspace(_lib.OP_ADD_RMS_NORM_GRAD, g2.shape[0], 0, g2.shape[1], 0, g2)
    _run(op, "qlin_add_rms_norm_grad", dy.device, g2, d2, h2, w, float(eps), _flat(dx), dw, ws.data_ptr() if ws is not None else 0,
         ws.numel() if ws is not None else 0)
    return dx, dw


def gated_act(gate, up=None, *, act="silu"):
    """f(gate) * up (up None: f(gate)) in fp32 with one rounding; act "silu" or "gelu_tanh"."""
    op = "gated_act"
    _disabled(op)
    kind = _act(op, act)
    if ops._FAST is not None:
        try:
            return ops._FAST.gated_act(gate, up, kind)
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, gate, up)
    g2, u2 = _rows(op, gate, "gate"), _rows(op, up, "up", gate.shape)
    y = torch.empty(gate.shape, dtype=gate.dtype, device=gate.device)
    _run(op, "qlin_gated_act", gate.device, g2, u2, kind, _flat(y))
    return y


def gated_act_int8(gate, up=None, *, act="silu", convrot_groupsize=0):
    """(codes, scale): gated_act in 8 bits."""
    op = "gated_act_int8"
    _disabled(op)
    kind = _act(op, act)
    if ops._FAST is not None:
        try:
            return ops._FAST.gated_act_int8(gate, up, kind, int(convrot_groupsize))
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, gate, up)
    g2, u2 = _rows(op, gate, "gate"), _rows(op, up, "up", gate.shape)
    q, scale = _codes(gate.shape, gate.device)
    _run(op, "qlin_gated_act_int8", gate.device, g2, u2, kind, int(convrot_groupsize), _flat(q), _flat(scale))
    return q, scale


def gated_act_grad(dy, gate, up=None, *, act="silu"):
    """(dgate, dup) of gated_act from the gradient of its output (dup None without up): the two halves of one tensor [.., 2
    values], which is the gradient of a fused projection's output."""
    op = "gated_act_grad"
    _disabled(op)
    kind = _act(op, act)
    if ops._FAST is not None:
        try:
            return ops._FAST.gated_act_grad(dy, gate, up, kind)
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, dy, gate, up)
    d2, g2, u2 = _rows(op, dy, "dy", gate.shape), _rows(op, gate, "gate"), _rows(op, up, "up", gate.shape)
    n = gate.shape[-1]
    both = torch.empty((*gate.shape[:-1], n if up is None else 2 * n), dtype=gate.dtype, device=gate.device)
    flat = _flat(both)
    _run(op, "qlin_gated_act_grad", gate.device, d2, g2, u2, kind, flat[:, :n], None if up is None else flat[:, n:])
    return (both, None) if up is None else (both[..., :n], both[..., n:])


def w8a8_int8_linear(x, x_scale, qdata, scale, bias=None, out_dtype=None, *, residual=None, residual_scale=None):
    """y = x_scale * scale * (x @ qdata^T) + bias over int8 rows x [.., K] with x_scale [.., 1] (quantize_int8_rowwise,
    add_rms_norm_int8, gated_act_int8) and int8 weights qdata [N, K] with scale [N], [N, 1] or a single element.  With `residual`
    ([.., N]): y = residual + residual_scale * that, one rounding.  out_dtype None: the residual's, else bf16."""
    op = "w8a8_int8_linear"
    _disabled(op)
    if ops._FAST is not None:
        try:
            return ops._FAST.w8a8_int8_linear(x, x_scale, qdata, scale, bias, out_dtype, residual, residual_scale)
        except ops._FastError as e:
            raise _fast_error(op, e) from None
    _check_device(op, x, x_scale, qdata, scale, bias, residual, residual_scale)
    _dtype(op, x, "x", torch.int8)
    _dtype(op, qdata, "qdata", torch.int8)
    x2 = _rows(op, x, "x")
    if qdata.dim() != 2:
        raise NoCapableBackendError(op, {"hip": "qdata must be a 2-D int8 tensor"})
    m, k = x2.shape
    n = qdata.shape[0]
    if x_scale.numel() != m:
        raise ValueError(f"{op}: x_scale has {x_scale.numel()} elements, expected {m}")
    if scale.numel() not in (1, n):
        raise ValueError(f"{op}: scale has {scale.numel()} elements, expected {n}")
    shape = (*x.shape[:-1], n)
    res = _residual_args(op, residual, residual_scale, shape, n)
    dt = out_dtype or (torch.bfloat16 if residual is None else residual.dtype)
    if dt not in ops._FLOAT:
        raise NoCapableBackendError(op, {"hip": f"out_dtype {dt} unsupported"})
    y = torch.empty(shape, dtype=dt, device=x.device)
    w = qdata if qdata.shape[1] <= 1 or qdata.stride(1) == 1 else qdata.contiguous()
    ws = _scale(scale, n)
    r, rs = res if res is not None else (None, None)
    xs = ops._f32_1d(x_scale)
    b = ops._bias(bias, n)
    param = (0 if k % 16 or _aligned(x2) else _lib.W8A8_X_ROWS) | (0 if k % 16 or _aligned(w) else _lib.W8A8_W_ROWS) | (
        0 if n <= 1 or w.stride(0) == k else _lib.W8A8_W_APART)
    room = ops._workspace(_lib.OP_W8A8_LINEAR, m, n, k, param, x2)
    _run(op, "qlin_w8a8_linear", x.device, x2, xs, w, ws, b, r, rs, _flat(y), room.data_ptr(), room.numel())
    return y


def _scale(scale, n):
    s = ops._f32_1d(scale)
    return s if s.numel() == n else s.expand(n).contiguous()


def _aligned(t):
    return t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or (t.stride(0) % 16 == 0 and t.stride(0) < 1 << 24))


# ------------------------------------------------------------------------------------------------
# Training
# ------------------------------------------------------------------------------------------------

class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h = add_rms_norm(x, residual, weight, eps=eps)
        ctx.save_for_backward(h, weight)
        ctx.conf = (float(eps), x.dtype)
        ctx.set_materialize_grads(False)
        return (y, None) if residual is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        h, weight = ctx.saved_tensors
        eps, dtype = ctx.conf
        need = ctx.needs_input_grad
        dx, dw = (dh, None) if dy is None else add_rms_norm_grad(dy, dh, h, weight, eps=eps, weight_grad=need[2])
        return dx.to(dtype) if need[0] and dx is not None else None, dx if need[1] else None, dw, None


class _GatedAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, act, packed):
        ctx.conf = (act, packed)
        ctx.save_for_backward(gate, up)
        if packed:
            gate, up = _halves(gate)
        return gated_act(gate, up, act=act)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        gate, up = ctx.saved_tensors
        act, packed = ctx.conf
        if packed:
            gate, up = _halves(gate)
            dgate, _ = gated_act_grad(dy, gate, up, act=act)
            return dgate._base, None, None, None
        dgate, dup = gated_act_grad(dy, gate, up, act=act)
        need = ctx.needs_input_grad
        return dgate if need[0] else None, dup if need[1] else None, None, None


def _halves(both):
    if both.shape[-1] % 2:
        raise ValueError(f"gated_act: rows of {both.shape[-1]} values have no halves")
    return both.chunk(2, -1)


class _W8A8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, qdata, scale, bias, convrot, convrot_groupsize):
        ctx.save_for_backward(qdata, scale)
        ctx.conf = (bool(convrot), int(convrot_groupsize), x.dtype)
        codes, x_scale = quantize_int8_rowwise(x, int(convrot_groupsize) if convrot else 0)
        return w8a8_int8_linear(codes, x_scale, qdata, scale, bias, x.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        qdata, scale = ctx.saved_tensors
        convrot, g, dtype = ctx.conf
        dx = None
        if ctx.needs_input_grad[0]:
            dx = int8_linear_grad_input(dy.contiguous(), qdata, scale, convrot, g, out_dtype=dtype)
        return dx, None, None, None, None, None


def add_rms_norm_trainable(x, residual=None, weight=None, eps=1e-6):
    """add_rms_norm with gradients for x, the residual and the weight (a frozen weight's is not formed); first derivatives
    only.  They are taken at h as it was stored (add_rms_norm_grad), which is kept for them in place of x and the residual."""
    y, h = _AddRmsNorm.apply(x, residual, weight, eps)
    return y, x if residual is None else h


def gated_act_trainable(gate, up=None, act="silu", packed=False):
    """gated_act with gradients for gate and up; first derivatives only.  packed: `gate` holds gate and up as the halves of its
    rows (a fused projection's output), and so does its gradient."""
    if packed and up is not None:
        raise ValueError("gated_act: packed rows hold up already")
    return _GatedAct.apply(gate, up, act, bool(packed))


def w8a8_linear_trainable(x, qdata, scale, bias=None, convrot=False, convrot_groupsize=256):
    """The linear over int8 rows of x (quantize_int8_rowwise, rotated with convrot) with an activation gradient: that of the
    linear over x itself, the rounding passed through (the weight, scale and bias stay frozen)."""
    return _W8A8Linear.apply(x, qdata, scale, bias, convrot, convrot_groupsize)
