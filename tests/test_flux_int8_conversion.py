"""``quantize_flux_model`` changes a model as a whole or not at all.  No GPU: the layers
are stand-ins."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch


class _Stub(torch.nn.Module):
    """In place of ``Int8Linear``; ``left`` of them can be made."""

    left = 0

    def __init__(self, linear=None):
        super().__init__()
        if _Stub.left == 0:
            raise torch.cuda.OutOfMemoryError("no memory")
        _Stub.left -= 1

    @classmethod
    def joined(cls, linears):
        return cls()


class _OnCuda(torch.nn.Module):
    weight = SimpleNamespace(is_cuda=True)


def _model(**kw):
    from hilberta_b200.flux_model import FluxTransformer

    model = FluxTransformer(num_double=2, num_single=2, dim=64, heads=2, head_dim=32, axes=(8, 12, 12), text_dim=16,
                            pooled_dim=8, device="cpu", **kw)
    model.x_embedder = _OnCuda()
    return model


@pytest.mark.parametrize("made", [0, 1, 5, 10, 22, 23, 25])
def test_failure_part_of_the_way(made, monkeypatch):
    from hilberta_b200 import flux_int8

    monkeypatch.setattr(flux_int8, "Int8Linear", _Stub)
    model = _model()
    before = dict(model.named_modules())
    ops = model.ops
    _Stub.left = made
    with pytest.raises(torch.cuda.OutOfMemoryError):
        flux_int8.quantize_flux_model(model)
    assert dict(model.named_modules()) == before and model.ops is ops and not getattr(model, "int8", False)
    _Stub.left = 1000
    assert flux_int8.quantize_flux_model(model) is model and model.int8
    kinds = [m for name, m in model.named_modules() if ".ff_" in name or ".mod" in name or ".proj_" in name]
    assert not any(isinstance(m, torch.nn.Linear) for m in kinds)
    assert 1000 - _Stub.left == 2 * 10 + 2 * 4  # every projection once


def test_own_block_operations_are_not_replaced(monkeypatch):
    from hilberta_b200 import flux_int8
    from hilberta_b200.block_ops import NativeBlockOps

    class Own(NativeBlockOps):
        pass

    monkeypatch.setattr(flux_int8, "Int8Linear", _Stub)
    _Stub.left = 1000
    for ops in (Own(), object()):
        model = _model(block_ops=ops)
        with pytest.raises(ValueError, match="block_ops"):
            flux_int8.quantize_flux_model(model)
        assert model.ops is ops and isinstance(model.transformer_blocks[0].mod_img, torch.nn.Linear)
