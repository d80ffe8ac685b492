"""``Int8Linear`` as a module: casts, moves and reloads keep its codes, its 32-bit
scales and the 16-byte rows that products need.  No GPU."""

from __future__ import annotations

import copy
import io
from types import SimpleNamespace

import pytest
import torch

BF16, FP16 = torch.bfloat16, torch.float16


def _layer(n=5, k=37, dtype=BF16, bias=True):
    """A layer as ``Int8Linear(linear)`` leaves it, on the CPU."""
    from hilberta_b200.int8 import Int8Linear

    g = torch.Generator().manual_seed(n + k)
    pitch = -(-k // 16) * 16
    values = torch.randint(-127, 128, (n, pitch), dtype=torch.int8, generator=g)[:, :k]
    layer = Int8Linear.__new__(Int8Linear)
    torch.nn.Module.__init__(layer)
    layer._set(SimpleNamespace(values=values, scales=torch.rand(n, generator=g) * 1e-3, dtype=dtype),
               torch.randn(n, generator=g).to(dtype) if bias else None)
    return layer


def _check(layer, like, dtype):
    """The codes and scales of ``like``, rows on 16 bytes, standing in for ``dtype``."""
    assert layer.values.dtype == torch.int8 and layer.scales.dtype == torch.float32 and layer.dtype == dtype
    assert torch.equal(layer.values, like.values) and torch.equal(layer.scales, like.scales)
    assert layer.values.stride(0) % 16 == 0 and layer.values.stride(1) == 1
    assert (layer.bias is None) == (like.bias is None) and (layer.bias is None or layer.bias.dtype == dtype)


@pytest.mark.parametrize("k", [32, 37, 1001])
@pytest.mark.parametrize("bias", [True, False])
def test_casts_keep_scales_and_codes(k, bias):
    want = _layer(k=k, bias=bias)
    for cast, dtype in ((lambda m: m.to(FP16), FP16), (lambda m: m.half(), FP16), (lambda m: m.half().bfloat16(), BF16),
                        (lambda m: m.to("cpu", BF16), BF16), (lambda m: m.float(), BF16), (lambda m: m.double(), BF16),
                        (lambda m: m.float().to(FP16), FP16), (lambda m: m.type(FP16), FP16)):
        layer = cast(torch.nn.Sequential(_layer(k=k, bias=bias)))[0]
        _check(layer, want, dtype)
    layer = _layer(k=k, bias=bias).float()  # no 16-bit type: the bias keeps its own
    assert layer.bias is None or torch.equal(layer.bias, want.bias)


@pytest.mark.parametrize("k", [48, 37])
def test_copies_and_moves_keep_aligned_rows(k):
    want = _layer(k=k)
    _check(copy.deepcopy(want), want, BF16)
    moved = _layer(k=k)
    moved._apply(lambda t: t.clone(memory_format=torch.contiguous_format))  # as a move to another device lays it out
    _check(moved, want, BF16)
    empty = _layer(k=k).to("meta").to_empty(device="cpu")
    assert empty.values.shape == want.values.shape and empty.values.stride(0) % 16 == 0
    empty.load_state_dict(want.state_dict())
    _check(empty, want, BF16)


@pytest.mark.parametrize("assign", [False, True])
@pytest.mark.parametrize("bias", [True, False])
def test_reload(assign, bias):
    want = _layer(bias=bias)
    buf = io.BytesIO()
    torch.save({name: t.contiguous() for name, t in want.state_dict().items()}, buf)  # rows side by side in the file
    buf.seek(0)
    layer = _layer(bias=bias)
    layer.values.zero_()
    layer.load_state_dict(torch.load(buf), assign=assign)
    _check(layer, want, BF16)
    if bias:  # an assigned bias brings its type
        state = {name: t.half() if t.is_floating_point() else t for name, t in want.state_dict().items()}
        layer.load_state_dict(state, assign=assign)
        assert layer.scales.dtype == torch.float32 and layer.bias.dtype == layer.dtype == (FP16 if assign else BF16)


def test_features():
    layer = _layer(n=7, k=37)
    assert (layer.in_features, layer.out_features) == (37, 7)
    assert "in_features=37, out_features=7, bias=True" in repr(layer)
