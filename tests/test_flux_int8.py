"""Host-side checks of the 8-bit FLUX model.  No GPU."""

from __future__ import annotations

import pytest
import torch


def _small():
    from hilberta_b200.flux_model import FluxTransformer

    return FluxTransformer(num_double=1, num_single=1, dim=256, heads=2, device="meta")


def test_refusals():
    from hilberta_b200.flux_int8 import quantize_flux_model
    from hilberta_b200.flux_tp import shard_flux_model

    with pytest.raises(TypeError, match="FluxTransformer"):
        quantize_flux_model(torch.nn.Linear(4, 4))
    with pytest.raises(ValueError, match="CUDA"):
        quantize_flux_model(_small())
    sharded = _small()
    sharded.tp_world = 2
    with pytest.raises(ValueError, match="sharded"):
        quantize_flux_model(sharded)
    done = _small()
    done.int8 = True
    with pytest.raises(ValueError, match="already"):
        quantize_flux_model(done)
    with pytest.raises(ValueError, match="8 bits"):
        shard_flux_model(done)
