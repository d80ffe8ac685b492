"""8-bit products of rows near the ends of the 16-bit types' range: the results are
those of sum * x_scale * w_scale + bias wherever that fits, for every scale of a bf16
token and weights' scales below 2^104, and do not depend on the kernel that serves the
number of tokens.

The integer sum is exact.  Its conversion and two multiplications, one fused with the
bias, round by at most 2^-24 each of |product| + |bias|, the result by at most half a
step of its type (2^-8 for bf16).  Scales of tokens below 2^-102 are multiplied by 2^-24
into fp32's subnormals: the least, 2^-100 / 127, and a product with it are then within
2^-150, half a step, of 2^-131, together 2^-18 of the product."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _check(got, xc, xs, wc, ws, bias):
    acc = (xc.double() @ wc.double().t()) * (xs.double()[:, None] * ws.double())
    ref = acc + bias.double()
    err = (got.double() - ref).abs()
    step = torch.where(xs < 2.0**-102, 2.0**-18, 4 * 2.0**-24).double()[:, None]
    bound = ref.abs() * 2.0**-8 + step * (acc.abs() + bias.double().abs()) * (1 + 2.0**-8) + 2.0**-133
    past = ref.abs() >= torch.finfo(BF16).max  # infinite by the formula as well
    assert bool((err[~past] <= bound[~past]).all()), float((err - bound)[~past].max())
    assert got[~past].isfinite().all() and past.float().mean() < 0.5


@pytest.mark.parametrize("m,k,n", [(1, 4096, 515), (2, 3000, 1000), (3, 2048, 300), (9, 4096, 640), (40, 1000, 136), (100, 4096, 1024),
                                   (600, 4096, 1030), (2500, 512, 2560), (300, 14000, 1500), (1280, 9000, 4096)])
def test_large_and_small_scales(m, k, n):
    import hilberta_b200 as hb

    g = torch.Generator(device="cuda").manual_seed(m + n)
    codes = lambda r: torch.randint(-127, 128, (r, -(-k // 16) * 16), dtype=torch.int8, generator=g, device="cuda")[:, :k]  # noqa: E731
    x, w = codes(m), codes(n)
    x[:, ::2] = w[0, ::2]  # sums of a million and more with the first channel
    large, small = torch.finfo(BF16).max / 127, 2.0**-100 / 127
    bias = torch.zeros(n, dtype=BF16, device="cuda")
    for xs, ws in ((large, 1e-9), (1e30, 1e-4), (1e-9, 2.0**103), (1e-5, 2e31), (large, small), (small, 1e31),
                   (2.0**-102, 2.0**100), (1e-20, 1e18)):
        rows = hb.Int8Rows(x, torch.full((m,), xs, device="cuda"), BF16)
        weight = hb.Int8Rows(w, torch.full((n,), ws, device="cuda"), BF16)
        got = hb.int8_linear(rows, weight, bias)
        _check(got, x, rows.scales, w, weight.scales, bias)
        some = slice(m // 2, m // 2 + 2)
        assert torch.equal(hb.int8_linear(rows.row_slice(some.start, min(some.stop, m)), weight, bias), got[some])


@pytest.mark.parametrize("m", [1, 4, 20, 200, 3000])
def test_tokens_of_every_size_beside_each_other(m):
    """16-bit tokens whose sizes span the type's range, every one as if it were alone."""
    import hilberta_b200 as hb

    k, n = 1024, 768
    g = torch.Generator(device="cuda").manual_seed(m)
    size = 2.0 ** torch.linspace(-110, 120, m, device="cuda")[:, None] if m > 1 else 2.0**118
    x = (torch.randn(m, k, generator=g, device="cuda") * size).to(BF16)
    w = hb.quantize_rows((1e-6 * torch.randn(n, k, generator=g, device="cuda")).to(BF16))
    rows, bias = hb.quantize_rows(x), torch.zeros(n, dtype=BF16, device="cuda")
    got = hb.int8_linear(x, w, bias)
    _check(got, rows.values, rows.scales, w.values, w.scales, bias)
    for i in (0, m // 2, m - 1):
        assert torch.equal(hb.int8_linear(x[i : i + 1], w, bias), got[i : i + 1])
