"""Activations held in 8 bits between the forward and the backward pass.

The reference keeps the int8 copy that a quantized GEMM made of its input (cuda/QLinear.py:34), with one scale for
the whole tensor, and computes the forward pass on it.  A checkpoint here is only what is *kept*: the forward pass
runs on the tensor itself, the backward pass on its 8-bit form, with one scale per run of columns of a row, so a row
of small values is not held at the resolution of the largest row.

    p = pack(x, group=32)                       # int8 values + fp32 scales: 1.125 bytes an element
    y = unpack(p)                               # the values it holds, in x's type
"""
import contextlib

import torch

from .kernels import _L, _current_device, _ptr, _stream, check

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
    [rows, ceil(cols / group)], and the ``shape`` and ``dtype`` of the tensor it stands for."""

    __slots__ = ("values", "scale", "group", "shape", "dtype")

    def __init__(self, values, scale, group, shape, dtype):
        self.values, self.scale, self.group, self.shape, self.dtype = values, scale, group, tuple(shape), dtype

    @property
    def device(self):
        return self.values.device

    def nbytes(self):
        return self.values.size(0) * self.values.stride(0) + 4 * self.scale.numel() if self.values.numel() else 0


def _rows_of(x):
    """[rows, cols] with contiguous columns: a view where x's layout allows one."""
    cols = x.size(-1)
    rows = x.numel() // cols if cols else 0
    if cols > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    return x.reshape(rows, cols)


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
        flat = _rows_of(x.detach())
        rows = flat.size(0)
        ld = (cols + 15) // 16 * 16
        values = torch.empty((rows, ld), dtype=torch.int8, device=x.device)[:, :cols]
        scale = torch.empty((rows, -(-cols // group)), dtype=torch.float32, device=x.device)
        check(_L.tango_pack_i8(_ptr(values), ld, _ptr(scale), _ptr(flat), DTYPES[x.dtype], rows, cols,
                               flat.stride(0) if rows > 1 else cols, group, _stream()), "pack")
    return Packed(values, scale, group, x.shape, x.dtype)


def unpack(packed, dtype=None):
    """The tensor that ``packed`` stands for: value * scale in fp32, rounded to ``dtype`` (default: the type of the
    tensor that was packed)."""
    if not isinstance(packed, Packed):
        raise TypeError("unpack: expected what pack returned")
    dtype = packed.dtype if dtype is None else dtype
    if dtype not in DTYPES:
        raise RuntimeError("unpack: expected torch.float32, torch.bfloat16 or torch.float16 but got %s" % dtype)
    with on_device_of(packed.values):
        out = torch.empty(packed.shape, dtype=dtype, device=packed.device)
        rows, cols = packed.values.shape
        check(_L.tango_unpack_i8(_ptr(out), DTYPES[dtype], cols, _ptr(packed.values), packed.values.stride(0),
                                 _ptr(packed.scale), rows, cols, packed.group, _stream()), "unpack")
    return out
