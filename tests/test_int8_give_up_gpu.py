"""8-bit products whose barrier waits run out: the launch reports it, writes right
outputs or none, leaves nothing under way, and the next one is whole again."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# tokens, inner size, channels: single CTAs of every width, alone and sharing K; CTA pairs
# that walk over tiles; two and four pairs on one tile's K; a last round in a launch of its own
SIZES = [(10, 128, 200), (10, 4096, 256), (30, 1024, 640), (60, 100, 1000), (60, 8192, 128), (128, 512, 1024), (200, 640, 2048),
         (4096, 512, 4096), (500, 9001, 3080), (260, 14000, 1500), (1280, 9000, 4096)]


@pytest.fixture
def limit():
    from hilberta_b200 import _lib

    lib = _lib.lib()
    yield lambda ms: _lib.check(lib.hb_int8_set_wait_limit(ms), "hb_int8_set_wait_limit")
    assert lib.hb_int8_set_wait_limit(2000) == 0


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("coded", [True, False])
def test_waits_that_run_out(m, k, n, coded, limit):
    import hilberta_b200 as hb
    from hilberta_b200 import _lib

    g = torch.Generator(device="cuda").manual_seed(m + n)
    x, w = ((torch.randn(r, k, generator=g, device="cuda")).to(torch.bfloat16) for r in (m, n))
    w = hb.quantize_rows(w)
    x = hb.quantize_rows(x) if coded else x
    want = hb.int8_linear(x, w, activation="gelu_tanh")
    assert hb.device_status() == 0 and want.isfinite().all()
    for _ in range(5):
        limit(0)  # gives up half-way through the first tile
        outs = [torch.full_like(want, math.nan) for _ in range(3)]
        for out in outs:
            hb.int8_linear(x, w, activation="gelu_tanh", out=out)
        limit(2000)
        again = hb.int8_linear(x, w, activation="gelu_tanh")  # right behind them
        assert hb.device_status() == _lib.HB_DEV_TIMEOUT
        for out in outs:
            assert out.isnan().any() and bool((out.isnan() | (out == want)).all())
        assert torch.equal(again, want)
    assert torch.equal(hb.int8_linear(x, w, activation="gelu_tanh"), want) and hb.device_status() == 0
