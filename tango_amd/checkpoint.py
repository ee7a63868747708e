"""Activations held in 8 bits between the forward and the backward pass.

The reference keeps the int8 copy that a quantized GEMM made of its input (cuda/QLinear.py:34), with one scale for
the whole tensor, and computes the forward pass on it.  A checkpoint here is only what is *kept*: the forward pass
runs on the tensor itself, the backward pass on its 8-bit form, with one scale per run of columns of a row, so a row
of small values is not held at the resolution of the largest row.

    p = pack(x, group=32)                       # int8 values + fp32 scales: 1.125 bytes an element
    y = unpack(p)                               # the values it holds, in x's type
    dw, db = weight_grad(dy, p, want_bias=True) # of a linear layer whose input x was, without restoring x

``CheckpointLinear`` is a linear layer that keeps its input that way; ``tango_amd.graph_attention`` keeps queries, keys
and values that way when asked to.
"""
import contextlib
import math
import operator

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import Function, once_differentiable

from .kernels import _L, _current_device, _ptr, _stream, _workspace, check, refuse_capture

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # tango_dtype of include/tango_hip.h


def on_device_of(t):
    """Launches go to the current stream of the tensors' own device, whichever device is current."""
    return contextlib.nullcontext() if t.device.index == _current_device() else torch.cuda.device(t.device)


def need_float(t, name):
    """A floating GPU tensor of a type that the kernels take."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    if t.dtype not in DTYPES:
        raise RuntimeError("%s: expected torch.float32, torch.bfloat16 or torch.float16 but got %s" % (name, t.dtype))
    if not t.is_cuda:
        raise RuntimeError("%s must be on GPU" % name)
    return t


class Packed:
    """What ``pack`` returns: ``values`` int8 [rows, cols] (rows start 16-byte aligned), ``scale`` fp32
    [rows, ceil(cols / group)], and the ``shape`` and ``dtype`` of the tensor it stands for.  Parts of a user's own
    are checked here, once, and cannot be replaced afterwards."""

    __slots__ = ("_values", "_scale", "_group", "_shape", "_dtype")
    values, scale, group, shape, dtype = (property(operator.attrgetter(name)) for name in __slots__)

    def __init__(self, values, scale, group, shape, dtype):
        if values.dtype != torch.int8 or scale.dtype != torch.float32 or dtype not in DTYPES:
            raise RuntimeError("Packed: values must be int8, the scale fp32, and dtype fp32, bf16 or fp16")
        if not isinstance(group, int) or group < 1:
            raise RuntimeError("Packed: group must be a positive whole number")
        *lead, cols = shape
        rows = math.prod(lead)
        if values.shape != (rows, cols):
            raise RuntimeError("Packed: the values do not have the tensor's shape")
        if cols > 1 and values.stride(1) != 1 or scale.shape != (rows, -(-cols // group)) or not scale.is_contiguous():
            raise RuntimeError("Packed: needs contiguous columns and a contiguous scale per row and run")
        self._fill(values, scale, group, shape, dtype)

    def _fill(self, values, scale, group, shape, dtype):
        self._values, self._scale, self._group, self._shape, self._dtype = values, scale, group, tuple(shape), dtype
        return self

    @property
    def device(self):
        return self._values.device

    def nbytes(self):
        return self._values.size(0) * self._values.stride(0) + 4 * self._scale.numel() if self._values.numel() else 0


def need_packed(packed, name):
    """A checkpoint on one GPU (it may have been saved and loaded elsewhere)."""
    if not isinstance(packed, Packed):
        raise TypeError("%s: expected what pack returned" % name)
    if not packed._values.is_cuda or packed._scale.device != packed._values.device:
        raise RuntimeError("%s: the checkpoint must be on GPU" % name)
    return packed


def rows_of(x):
    """[rows, cols] with contiguous columns: a view where x's layout allows one."""
    cols = x.size(-1)
    rows = math.prod(x.shape[:-1])
    if cols > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    return x.reshape(rows, cols)


def pack_rows(x, group, scale):
    """The int8 values of a 2-D tensor with contiguous columns; its scales go into ``scale`` [rows, runs], any strides."""
    rows, cols = x.shape
    ld = (cols + 15) // 16 * 16
    values = torch.empty((rows, ld), dtype=torch.int8, device=x.device)[:, :cols]
    check(_L.tango_pack_i8(_ptr(values), ld, _ptr(scale), scale.stride(0), scale.stride(1), _ptr(x), DTYPES[x.dtype], rows, cols,
                           x.stride(0) if rows > 1 else cols, group, _stream()), "pack")
    return values


def pack(x, group=None):
    """The 8-bit form of ``x`` [..., cols] (fp32, bf16 or fp16 on the GPU): per run of ``group`` consecutive columns
    (None: the whole row; the last run of a row may be shorter) the scale max|x| / 127 and the integers nearest to
    127 x / max|x|, ties to even.  A run that holds an infinity or a NaN comes back as NaN throughout."""
    need_float(x, "x")
    if x.dim() < 1:
        raise RuntimeError("pack: x needs at least one dimension")
    cols = x.size(-1)
    if group is None:
        group = max(cols, 1)
    if int(group) != group or group < 1:
        raise ValueError("pack: group must be a positive whole number of columns")
    group = int(group)
    with on_device_of(x):
        flat = rows_of(x.detach())
        scale = torch.empty((flat.size(0), -(-cols // group)), dtype=torch.float32, device=x.device)
        values = pack_rows(flat, group, scale)
    return Packed.__new__(Packed)._fill(values, scale, group, x.shape, x.dtype)


def unpack(packed, dtype=None):
    """The tensor that ``packed`` stands for: value * scale in fp32, rounded to ``dtype`` (default: the type of the
    tensor that was packed)."""
    need_packed(packed, "unpack")
    dtype = packed.dtype if dtype is None else dtype
    if dtype not in DTYPES:
        raise RuntimeError("unpack: expected torch.float32, torch.bfloat16 or torch.float16 but got %s" % dtype)
    with on_device_of(packed.values):
        out = torch.empty(packed.shape, dtype=dtype, device=packed.device)
        rows, cols = packed.values.shape
        check(_L.tango_unpack_i8(_ptr(out), DTYPES[dtype], cols, _ptr(packed.values), packed.values.stride(0),
                                 _ptr(packed.scale), rows, cols, packed.group, _stream()), "unpack")
    return out


def weight_grad(dy, packed, want_bias=False):
    """``dy.T @ x`` (and, with ``want_bias``, ``dy.sum(0)``) for the x that ``packed`` holds: the gradients of a linear
    layer's weight [out, in] and bias from the gradient ``dy`` [..., out] of its output, in dy's type, read straight
    from the 8-bit values.  Sums are fp32 in a fixed order.  Where dy, or dy times a row's scale, is not a finite fp32
    number the result is not finite either (an infinity or a NaN)."""
    need_float(dy, "dy")
    need_packed(packed, "weight_grad")
    if dy.dim() < 1 or dy.device != packed.device:
        raise RuntimeError("weight_grad: dy must be [..., out] on the checkpoint's device")
    rows, cols = packed.values.shape
    n = dy.size(-1)
    if math.prod(dy.shape[:-1]) != rows:
        raise RuntimeError("weight_grad: dy needs a row for each of the checkpoint's %d" % rows)
    with on_device_of(dy):
        flat = rows_of(dy.detach())
        if rows == 0:
            dw, db = flat.new_zeros((n, cols)), flat.new_zeros(n)
        else:
            dw = torch.empty((n, cols), dtype=dy.dtype, device=dy.device)
            db = torch.empty(n, dtype=dy.dtype, device=dy.device) if want_bias else None
            if cols == 0 and want_bias:
                db = flat.float().sum(0).to(dy.dtype)
            ws_bytes = _L.tango_weight_grad_i8_workspace(DTYPES[dy.dtype], rows, n, cols, packed.group)
            ws = _workspace(ws_bytes, dy.device)
            check(_L.tango_weight_grad_i8(_ptr(dw), _ptr(db) if want_bias else None, _ptr(flat), DTYPES[dy.dtype],
                                          flat.stride(0) if rows > 1 else n, _ptr(packed.values), packed.values.stride(0),
                                          _ptr(packed.scale), packed.group, rows, n, cols, _ptr(ws), ws_bytes, _stream()),
                  "weight_grad")
    return (dw, db) if want_bias else dw


class checkpoint_linear(Function):
    """``x @ weight.T + bias`` on the tensors themselves, keeping x in 8 bits (``pack(x, group)``) for the weight's
    gradient.  The input's gradient dy @ weight does not need x."""

    @staticmethod
    def forward(ctx, x, weight, bias, group=None):
        if torch.is_autocast_enabled("cuda"):  # as F.linear does below, so that what is kept is what it ran on
            to = torch.get_autocast_dtype("cuda")
            x, weight, bias = (t.to(to) if isinstance(t, torch.Tensor) and t.dtype in DTYPES else t for t in (x, weight, bias))
        for t, name in ((x, "x"), (weight, "weight")) + (((bias, "bias"),) if bias is not None else ()):
            need_float(t, name)
            if t.dtype != x.dtype or t.device != x.device:
                raise RuntimeError("checkpoint_linear: %s must have x's type and device" % name)
        ctx.has_bias = bias is not None
        held = pack(x, group) if ctx.needs_input_grad[1] else None
        # saved and not kept on ctx: released with the backward pass, as what other layers save is
        ctx.held = held and (held.group, held.shape, held.dtype)
        ctx.save_for_backward(weight if ctx.needs_input_grad[0] else None, *((held.values, held.scale) if held else ()))
        return F.linear(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        refuse_capture("checkpoint_linear.backward")
        weight, *held = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dx = torch.matmul(dy, weight) if want_x else None
        dw = db = None
        if want_w:
            held = Packed.__new__(Packed)._fill(*held, *ctx.held)
            dw, db = weight_grad(dy, held, True) if want_b else (weight_grad(dy, held), None)
        elif want_b:
            db = dy.float().reshape(-1, dy.size(-1)).sum(0).to(dy.dtype)
        return dx, dw, db, None


class CheckpointLinear(nn.Linear):
    """``nn.Linear`` (same parameters and state dict) whose input is held in 8 bits between the passes, with a scale
    per run of ``group`` columns of a row (None: one a row).  Beside ``QLinear``: the forward pass and the input's
    gradient are not quantized, only what the weight's gradient reads is."""

    def __init__(self, in_features, out_features, bias=True, group=None, **kw):
        super().__init__(in_features, out_features, bias, **kw)
        if group is not None and (int(group) != group or group < 1):
            raise ValueError("CheckpointLinear: group must be a positive whole number of columns")
        self.group = group

    def forward(self, x):
        return checkpoint_linear.apply(x, self.weight, self.bias, self.group)
