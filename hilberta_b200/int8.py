"""Linear layers in 8-bit integers (``hb_quantize_rows``, ``hb_int8_linear``): weights
and activations as int8 codes with one fp32 scale per row (per output channel,
per token), products summed exactly in 32-bit integers.

``quantize_rows(x)``                  16-bit rows -> ``Int8Rows`` (weights and activations alike)
``quantize_rows(a, joined=b)``        the rows [a | b] without the concatenation
``int8_linear(x, weight, bias, ...)`` act((x @ weight^T) + bias) in 16 bits
``Int8Linear(linear)``                a ``torch.nn.Linear`` with 8-bit weights

A row's scale is max|x| / 127 and its codes round(x * (127 / max|x|)), ties to
even.  A row holding an infinity or NaN gets the scale NaN: every output made
from it is NaN.  Inference only, CUDA only.
"""

from __future__ import annotations

import torch

from . import _lib

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_ACTIVATIONS = {None: 0, "gelu_tanh": 1}
_MAX_ROWS = (1 << 31) - 1
_used: set = set()  # devices with int8 launches (read by paired_kernel.device_status)


def _row_stride(t):
    """Row stride of a [..., K] tensor whose rows are equally spaced; None if they are not."""
    if t.ndim == 2:
        return t.stride()[0]
    if t.ndim == 1:
        return t.shape[0]
    shape, strides = t.shape, t.stride()
    rs, want = None, None
    for d in range(t.ndim - 2, -1, -1):
        if shape[d] == 1:
            continue
        if want is None:
            rs = strides[d]
        elif strides[d] != want:
            return None
        want = strides[d] * shape[d]
    return t.shape[-1] if rs is None else rs


class Int8Rows:
    """A matrix in 8 bits: ``values`` int8 ``[..., K]`` and ``scales`` fp32 ``[...]``;
    row r stands for ``values[r] * scales[r]``.  ``dtype`` is the 16-bit type it
    stands in for (the output type of products).  Rows are equally spaced and
    start on 16-byte boundaries (``quantize_rows`` pads them)."""

    __slots__ = ("values", "scales", "dtype", "row_stride")

    def __init__(self, values, scales, dtype):
        if values.dtype != torch.int8 or scales.dtype != torch.float32:
            raise TypeError("int8 values and float32 scales required")
        if dtype not in _DTYPES:
            raise TypeError("dtype must be float16 or bfloat16")
        if not values.is_cuda or scales.device != values.device:
            raise ValueError("values and scales must be on the same CUDA device")
        if values.ndim < 1 or scales.shape != values.shape[:-1] or not scales.is_contiguous():
            raise ValueError("scales must be contiguous with one entry per row of values")
        rs = _row_stride(values)
        if values.shape[-1] > 1 and values.stride(-1) != 1:
            raise ValueError("values must have a contiguous last dimension")
        if scales.numel() <= 1:  # the stride of a single row is never used
            rs = -(-values.shape[-1] // 16) * 16
        if rs is None or rs % 16 or rs < values.shape[-1] or values.data_ptr() % 16:
            raise ValueError("rows of values must be equally spaced, 16-byte aligned and must not overlap")
        self.values, self.scales, self.dtype, self.row_stride = values, scales, dtype, rs

    @property
    def shape(self):
        return self.values.shape

    @property
    def device(self):
        return self.values.device

    @property
    def ndim(self):
        return self.values.ndim

    def dequantize(self):
        """The values in 16 bits (for checks; products never form them)."""
        return (self.values.float() * self.scales.unsqueeze(-1)).to(self.dtype)

    def row_slice(self, start, stop):
        """Rows [start, stop) of a 2-D matrix, sharing its storage (e.g. the output
        channels of one projection of a joined weight)."""
        if self.ndim != 2:
            raise ValueError("row_slice needs a 2-D matrix")
        return Int8Rows(self.values[start:stop], self.scales[start:stop], self.dtype)


def _empty_rows(shape, like):
    """Uninitialised ``Int8Rows`` of a shape, on the device and standing in for the type of ``like``."""
    *lead, K = shape
    pitch = -(-K // 16) * 16
    values = like.new_empty(*lead, pitch, dtype=torch.int8)  # (sizes one by one: a third faster than a tuple)
    rows = object.__new__(Int8Rows)  # right by construction: none of the checks of Int8Rows(...)
    rows.values = values if pitch == K else values[..., :K]
    rows.scales = like.new_empty(*lead, dtype=torch.float32) if lead else like.new_empty((), dtype=torch.float32)
    rows.dtype, rows.row_stride = like.dtype, pitch
    return rows


def _check_source(x, what):
    if not isinstance(x, torch.Tensor) or x.ndim < 1:
        raise TypeError(f"{what} must be a tensor of rows")
    if not x.is_cuda:
        raise ValueError("CUDA tensors required")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what} must be float16 or bfloat16")
    if x.shape[-1] < 1 or x.stride()[-1] != 1 and x.shape[-1] > 1:
        raise ValueError(f"{what} must have a nonempty contiguous last dimension")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("Inference only; disable autograd")


def quantize_rows(x, *, joined=None):
    """``Int8Rows`` of ``x`` (``[..., K]``, float16 or bfloat16, contiguous last
    dimension, rows equally spaced); with ``joined`` (``[..., Kj]``, same leading
    shape and type) of the rows ``[x | joined]``, one scale for both parts."""
    _check_source(x, "x")
    ka, kb, j_rs = x.shape[-1], 0, 0
    if joined is not None:
        _check_source(joined, "joined")
        if joined.shape[:-1] != x.shape[:-1] or joined.dtype != x.dtype or joined.device != x.device:
            raise ValueError("joined must match x's leading shape, dtype and device")
        kb, j_rs = joined.shape[-1], _row_stride(joined)
    x_rs = _row_stride(x)
    if x_rs is None or j_rs is None:
        raise ValueError("rows must be equally spaced")
    if ka + kb > _lib.HB_INT8_MAX_K:
        raise NotImplementedError(f"rows of more than {_lib.HB_INT8_MAX_K} values are not supported")
    rows = x.numel() // ka
    if rows > _MAX_ROWS:
        raise NotImplementedError("2^31 rows or more are not supported")
    out = _empty_rows((*x.shape[:-1], ka + kb), x)
    with _lib.on_device(x.device) as stream:
        rc = _lib.lib().hb_quantize_rows(
            x.data_ptr(), x_rs, ka, None if joined is None else joined.data_ptr(), j_rs, kb, rows, out.values.data_ptr(),
            out.row_stride, out.scales.data_ptr(), _DTYPES[x.dtype], stream)
    _lib.check(rc, "hb_quantize_rows")
    return out


def int8_linear(x, weight, bias=None, *, activation=None, out=None):
    """``act(x @ weight^T + bias)`` with both operands in 8 bits.

    ``x``: ``Int8Rows [..., K]``, or a 16-bit tensor ``[..., K]`` that is quantised
    in the call.  ``weight``: ``Int8Rows [N, K]``.  ``bias``: ``[N]`` in x's type or
    None.  ``activation``: None or ``"gelu_tanh"``.  ``out`` (allocated when not
    given): ``[..., N]`` in x's type with a contiguous last dimension; rows may be
    spaced (a slice of a wider buffer), a leading dimension whose rows are not
    equally spaced takes one launch per index.  Integer sums are exact, so equal
    inputs give equal outputs whatever the number of tokens.  Results are
    ``(sum * x_scale) * weight_scale + bias`` in fp32, rounded once; weight scales must
    be below 2^104 (weights below 2.5e33), tokens may reach their type's end."""
    if not isinstance(weight, Int8Rows) or weight.values.ndim != 2:
        raise TypeError("weight must be 2-D Int8Rows [N, K] (quantize_rows of a weight matrix)")
    coded = isinstance(x, Int8Rows)
    if coded:
        x_shape = x.values.shape
    else:
        _check_source(x, "x")
        x_shape = x.shape
    N, K = weight.values.shape
    kind, dev = x.dtype, x.device
    if x_shape[-1] != K:
        raise ValueError("x and weight must have the same inner size")
    if N > _MAX_ROWS or (x.scales.numel() if coded else x.numel() // K) > _MAX_ROWS:
        raise NotImplementedError("2^31 rows or more are not supported")
    if weight.values.device != dev:
        raise ValueError("x and weight must be on the same CUDA device")
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError('activation must be None or "gelu_tanh"')
    if bias is not None:
        if bias.shape != (N,) or bias.dtype != kind or bias.device != dev or not bias.is_contiguous():
            raise ValueError("bias must be a contiguous [N] tensor of x's type and device")
        if bias.requires_grad and torch.is_grad_enabled():
            raise ValueError("Inference only; disable autograd")
    shape = (*x_shape[:-1], N)
    if out is None:
        out = (x.values if coded else x).new_empty(*shape, dtype=kind)
    else:
        if out.shape != shape or out.dtype != kind or out.device != dev or (N > 1 and out.stride(-1) != 1):
            raise ValueError("out must be [..., N] of x's type and device with a contiguous last dimension")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("Inference output cannot require gradients")
        _check_out(out, x, weight, bias)
    _product(x, coded, weight, bias, act, out, kind, dev)
    return out


def _check_out(out, x, weight, bias):
    if _overlaps_itself(out):
        raise ValueError("out must not overlap itself")
    parts = [x.values, x.scales] if isinstance(x, Int8Rows) else [x]
    for t in (*parts, weight.values, weight.scales, bias):
        if t is not None and not _apart(out, t):
            raise ValueError("out cannot alias inputs")


def _overlaps_itself(t):
    reach = 0
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if st <= reach:
            return True
        reach += st * (n - 1)
    return False


def _span(t):
    if t.numel() == 0:
        return t.data_ptr(), t.data_ptr()
    extent = sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1
    return t.data_ptr(), t.data_ptr() + extent * t.element_size()


def _apart(a, b):
    """No element of a is one of b: their memory ranges are apart, or both are rows of
    one spacing that lie side by side (column slices of one buffer)."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return True
    ra, rb = _row_stride(a), _row_stride(b)
    if ra is None or rb is None or a.ndim < 2 or b.ndim < 2:
        return False
    pitch = ra * a.element_size()
    wa, wb = a.shape[-1] * a.element_size(), b.shape[-1] * b.element_size()
    if pitch != rb * b.element_size() or pitch <= 0:
        return False
    shift = (b0 - a0) % pitch
    return shift >= wa and shift + wb <= pitch


def _product(x, coded, weight, bias, act, out, kind, dev):
    out_rs = _row_stride(out)
    x_rs = x.row_stride if coded else _row_stride(x)
    if out_rs is None or x_rs is None:  # a leading index at a time
        for i in range(out.shape[0]):
            part = Int8Rows(x.values[i], x.scales[i], x.dtype) if coded else x[i]
            _product(part, coded, weight, bias, act, out[i], kind, dev)
        return
    lib = _lib.lib()
    w = weight.values
    N, K = w.shape
    M = x.scales.numel() if coded else x.numel() // K
    tail = (w.data_ptr(), weight.row_stride, weight.scales.data_ptr(), None if bias is None else bias.data_ptr(),
            out.data_ptr(), out_rs, M, N, K, act, _DTYPES[kind])
    with _lib.on_device(dev) as stream:
        if coded:
            rc = lib.hb_int8_linear(x.values.data_ptr(), x_rs, x.scales.data_ptr(), *tail, stream)
        else:
            nbytes = lib.hb_int8_linear16_workspace_bytes(M, K)
            ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
            rc = lib.hb_int8_linear16(x.data_ptr(), x_rs, *tail, None if ws is None else ws.data_ptr(), nbytes, stream)
    if rc == 0:
        _used.add(dev.index)
        return
    if rc == _lib.HB_ERR_UNSUPPORTED:
        raise NotImplementedError(f"int8_linear: {_lib.status_text(rc)}")
    _lib.check(rc, "hb_int8_linear")


def _aligned_rows(values):
    """[N, K] codes whose rows start on 16-byte boundaries: as they are, or a copy
    (moving a tensor to another device lays its rows side by side)."""
    N, K = values.shape
    if N <= 1 or (values.stride(0) % 16 == 0 and (K == 1 or values.stride(1) == 1)):
        return values
    return values.new_empty(N, -(-K // 16) * 16)[:, :K].copy_(values)


class Int8Linear(torch.nn.Module):
    """``torch.nn.Linear`` with 8-bit weights, quantised once from ``linear`` (a
    CUDA layer in float16 or bfloat16): y = int8_linear(x, weight, bias).

    ``forward`` takes 16-bit tensors or ``Int8Rows``.  ``weight`` is the layer's
    ``Int8Rows``; its parts are the buffers ``values`` and ``scales``.  Casts of the
    module change the 16-bit type that it stands in for and the bias, never codes and
    scales; a cast to another type than those leaves the layer as it is."""

    def __init__(self, linear):
        super().__init__()
        self._set(quantize_rows(linear.weight.detach()), None if linear.bias is None else linear.bias.detach())

    def _set(self, rows, bias):
        self.dtype = rows.dtype
        self.register_buffer("values", rows.values)
        self.register_buffer("scales", rows.scales)
        self.register_buffer("bias", bias)

    def _apply(self, fn, recurse=True):
        values, scales, bias = self.values, self.scales, self.bias
        super()._apply(fn, recurse)
        device = self.scales.device
        if self.scales.dtype in _DTYPES:  # a cast
            self.dtype = self.scales.dtype
        elif bias is not None and self.bias.dtype != self.dtype:
            self.bias = bias.to(device)
        if self.scales.dtype != torch.float32:
            self.scales = scales.to(device)
        self.values = _aligned_rows(self.values if self.values.dtype == torch.int8 else values.to(device))
        return self

    def _load_from_state_dict(self, *args):
        super()._load_from_state_dict(*args)  # assign=True: the buffers are the file's own tensors
        self.values, self.scales = _aligned_rows(self.values), self.scales.float()
        if self.bias is not None and self.bias.dtype in _DTYPES:
            self.dtype = self.bias.dtype

    @property
    def in_features(self):
        return self.values.shape[1]

    @property
    def out_features(self):
        return self.values.shape[0]

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"dtype={self.dtype}")

    @classmethod
    def joined(cls, linears):
        """One layer of several that read the same input: their outputs side by side."""
        self = cls.__new__(cls)
        torch.nn.Module.__init__(self)
        weight = torch.cat([m.weight.detach() for m in linears])
        bias = None
        if any(m.bias is not None for m in linears):
            bias = torch.cat([weight.new_zeros(m.weight.shape[0]) if m.bias is None else m.bias.detach() for m in linears])
        self._set(quantize_rows(weight), bias)
        return self

    def outputs(self, start, stop):
        """The layer of output channels [start, stop), sharing this one's storage."""
        part = Int8Linear.__new__(Int8Linear)
        torch.nn.Module.__init__(part)
        part._set(self.weight.row_slice(start, stop), None if self.bias is None else self.bias[start:stop])
        return part

    @property
    def weight(self):
        return Int8Rows(self.values, self.scales, self.dtype)

    def forward(self, x, *, activation=None, out=None):
        return int8_linear(x, self.weight, self.bias, activation=activation, out=out)


__all__ = ["Int8Rows", "Int8Linear", "quantize_rows", "int8_linear"]
