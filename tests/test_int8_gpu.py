"""8-bit linear layers (hilberta_b200/int8.py, the int8 forms of block_ops) against
their formulas in 64 bits.

Row quantisation is elementwise, correctly rounded fp32 arithmetic, so codes and
scales are compared exactly.  A product's integer sum is exact; what follows is fp32:
converting the sum, two scale multiplications (one fused with the bias) round
four times, each by at most 2^-24 of |product| + |bias|, and the result once to
16 bits, by at most eps/2 of itself.  tanh-GELU has slope at most 1.13, and its
own fp32 steps stay within 2^-18 of the result: the exponent's three roundings
are magnified by |exponent| * ln 2 <= 20 where the result is not negligible.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(m, k, dtype, seed, spread=1.0):
    g = _gen(seed)
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp(spread * torch.randn(k, generator=g, device="cuda"))
    return x.to(dtype)


def _quantised(x):
    """(codes, scales) of the rows of x by the definition: each fp32 operation as the
    64-bit one rounded to fp32, which is the same (products of two fp32 numbers are
    exact in 64 bits, and a 64-bit quotient rounds to the correctly rounded one)."""
    f = x.double()
    top = f.abs().amax(-1)
    live = (top >= 2.0**-100) & torch.isfinite(top)
    inv = torch.where(live, 127 / top, 0.0).float().double()
    scale = torch.where(live, (top / 127).float(), torch.where(top < 2.0**-100, 0.0, math.nan))
    codes = torch.where(live[..., None], torch.round((f * inv[..., None]).float()), 0.0)
    return codes.to(torch.int8), scale


def _gelu64(v):
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v**3)))


def _check_product(got, xc, xs, wc, ws, bias, act):
    acc = (xc.double() @ wc.double().t()) * (xs.double()[:, None] * ws.double())
    b = 0.0 if bias is None else bias.double()
    ref = acc + b
    slack = 4 * 2.0**-24 * (acc.abs() + (b.abs() if bias is not None else 0.0))
    rel = torch.finfo(got.dtype).eps / 2
    if act:
        slack, rel, ref = 1.13 * slack + 1e-9, rel + 2.0**-18, _gelu64(ref)
    tiny = 2.0**-25 if got.dtype == FP16 else 0.0  # half a step of the subnormals
    err = (got.double() - ref).abs()
    bound = ref.abs() * rel + slack * (1 + rel) + tiny
    assert bool((err <= bound).all()), (float((err - bound).max()), int((err > bound).sum()))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (5, 8), (130, 768), (64, 1001), (33, 2048), (17, 2056), (9, 8192),
                                 (6, 15360), (2, 33000), (2, 131072)])
def test_quantize_rows_is_exact(m, k, dtype):
    import hilberta_b200 as hb

    x = _rows(m, k, dtype, seed=k + m)
    got = hb.quantize_rows(x)
    codes, scales = _quantised(x)
    assert torch.equal(got.values, codes) and torch.equal(got.scales, scales)
    assert got.shape == (m, k) and got.dtype == dtype and got.values.data_ptr() % 16 == 0
    # half a step from the value, and the rounding of x * inv (2^-24 of at most 127 steps)
    off = (got.values.double() * got.scales.double()[:, None] - x.double()).abs()
    assert bool((off <= got.scales.double()[:, None] * (0.5 + 127 * 2.0**-22)).all())


def test_quantize_rows_strides_joined_and_leading_shape():
    import hilberta_b200 as hb

    big = _rows(40, 700, BF16, seed=1)
    for view in (big[:, 4:300], big[::2, 8:264], big.view(4, 10, 700)[:, :, :64]):  # 8-byte offset, row step 2, 3-D
        got = hb.quantize_rows(view)
        codes, scales = _quantised(view)
        assert torch.equal(got.values, codes) and torch.equal(got.scales, scales)
    for ka, kb in ((256, 1024), (5, 12), (3072, 12288), (9, 130)):
        a, b = _rows(21, ka, FP16, seed=2), _rows(21, kb, FP16, seed=3, spread=1.5)
        got = hb.quantize_rows(a, joined=b)
        codes, scales = _quantised(torch.cat([a, b], 1))
        assert torch.equal(got.values, codes) and torch.equal(got.scales, scales)
    one = hb.quantize_rows(big[7])
    assert one.values.shape == (700,) and one.scales.shape == ()
    assert hb.quantize_rows(big[:0]).values.shape == (0, 700)


@pytest.mark.parametrize("k", [64, 3000, 20000])
def test_quantize_rows_special_values(k):
    import hilberta_b200 as hb

    x = _rows(8, k, BF16, seed=5)
    x[0] = 0
    x[1, k // 2] = math.inf
    x[2, 0] = math.nan
    x[3, -1] = -math.inf
    x[4] = 1e-35  # below 2^-100
    x[5] = torch.finfo(BF16).max
    x[6] = -x[6].abs()
    got = hb.quantize_rows(x)
    codes, scales = _quantised(x)
    assert torch.equal(got.values, codes)
    assert torch.equal(got.scales.nan_to_num(-1.0), scales.nan_to_num(-1.0))
    assert got.scales[0] == 0 and got.scales[1:4].isnan().all() and got.scales[4] == 0
    # their products: the bias alone for zero rows, NaN for rows that held a non-finite value
    w = hb.quantize_rows(_rows(48, k, BF16, seed=6))
    bias = _rows(1, 48, BF16, seed=7)[0]
    out = hb.int8_linear(got, w, bias)
    assert torch.equal(out[0], bias) and torch.equal(out[4], bias)
    assert out[1:4].isnan().all() and out[6:].isfinite().all()
    assert not out[5].isnan().any()  # K values of 3.4e38 each: sums past the type's range are infinite


SIZES = [(1, 1, 1), (1, 64, 16), (2, 768, 3072), (3, 130, 127), (4, 4096, 1000), (5, 1000, 300), (7, 65, 9), (8, 512, 256),
         (16, 3072, 1280), (65, 1001, 129), (127, 128, 128), (128, 2048, 64), (129, 136, 1333), (256, 640, 256),
         (257, 1024, 260), (300, 5000, 384), (512, 3072, 1024), (1000, 100, 2048), (1771, 1001, 1333), (2500, 384, 2560),
         (4173, 512, 3000)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dtype,bias,act", [(BF16, True, None), (FP16, False, "gelu_tanh")])
def test_int8_linear(m, k, n, dtype, bias, act):
    import hilberta_b200 as hb

    x = _rows(m, k, dtype, seed=m + k + n, spread=0.5)
    w = hb.quantize_rows((_rows(n, k, dtype, seed=11, spread=0.0) / math.sqrt(k)).to(dtype))
    b = _rows(1, n, dtype, seed=12)[0] if bias else None
    got = hb.int8_linear(x, w, b, activation=act)
    codes, scales = _quantised(x)
    assert got.shape == (m, n) and got.dtype == dtype
    _check_product(got, codes, scales, w.values, w.scales, b, act)
    assert torch.equal(hb.int8_linear(hb.quantize_rows(x), w, b, activation=act), got)
    assert hb.device_status() == 0


def test_int8_linear_extreme_codes_are_exact():
    """Sums up to 127 * 127 * K: every product 127 * +-127, in types that hold the result's leading bits."""
    import hilberta_b200 as hb

    for m, k, n in ((2, 131072, 256), (200, 131072, 144)):
        x = torch.full((m, k), 127, dtype=torch.int8, device="cuda")
        w = torch.full((n, k), 127, dtype=torch.int8, device="cuda")
        w[1::2] = -127
        w[:, ::3] = 5
        rows = hb.Int8Rows(x, torch.full((m,), 2.0**-16, device="cuda"), BF16)
        weight = hb.Int8Rows(w, torch.ones(n, device="cuda"), BF16)
        _check_product(hb.int8_linear(rows, weight), x, rows.scales, w, weight.scales, None, None)


@pytest.mark.parametrize("m", [3, 200, 2000])
def test_int8_linear_out_views_and_neighbours(m):
    """Rows of a wider buffer: the columns around them stay as they are."""
    import hilberta_b200 as hb

    k, n = 384, 520
    x, w = _rows(m, k, BF16, seed=1), hb.quantize_rows(_rows(n, k, BF16, seed=2))
    want = hb.int8_linear(x, w)
    for left, width in ((0, 1024), (8, 1024), (3, 1001), (1, 530)):  # aligned, offset, odd row pitch, odd offset
        buf = torch.full((m + 2, width), 7.0, dtype=BF16, device="cuda")
        out = buf[1:m + 1, left:left + n]
        assert hb.int8_linear(x, w, out=out) is out
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert bool((buf == 7.0).all())
    # a batch whose rows are not equally spaced
    x3 = _rows(2 * m, k, BF16, seed=3).view(2, m, k)
    buf = torch.full((2, m + 5, n), 7.0, dtype=BF16, device="cuda")
    hb.int8_linear(x3, w, out=buf[:, 5:])
    assert torch.equal(buf[:, 5:], hb.int8_linear(x3, w)) and bool((buf[:, :5] == 7.0).all())


def test_int8_linear_empty_and_one():
    import hilberta_b200 as hb
    from hilberta_b200.block_ops import adaln_int8

    w = hb.quantize_rows(_rows(40, 64, BF16, seed=1))
    x = _rows(6, 64, BF16, seed=2)
    assert hb.int8_linear(x[:0], w).shape == (0, 40) and hb.int8_linear(hb.quantize_rows(x[:0]), w).shape == (0, 40)
    assert hb.int8_linear(x, w.row_slice(0, 0)).shape == (6, 0)
    want = hb.int8_linear(x, w)
    assert torch.equal(hb.int8_linear(x[3], w), want[3]) and torch.equal(hb.int8_linear(x.view(2, 3, 64), w), want.view(2, 3, 40))
    assert torch.equal(hb.int8_linear(x, w.row_slice(7, 8)), want[:, 7:8])
    m = torch.zeros(1, 256, dtype=BF16, device="cuda")
    assert adaln_int8(torch.zeros(1, 0, 256, dtype=BF16, device="cuda"), m, m).shape == (1, 0, 256)


def test_int8_linear_more_tokens_than_grid_rows():
    """8.4 million tokens: past 65535 tiles of 128, outputs past 2^31 bytes."""
    import hilberta_b200 as hb

    m, k, n = 8_400_003, 16, 136
    x = torch.randint(-127, 128, (m, k), dtype=torch.int8, device="cuda", generator=_gen(1))
    rows = hb.Int8Rows(x, torch.full((m,), 0.5, device="cuda"), BF16)
    w = hb.quantize_rows(_rows(n, k, BF16, seed=2))
    got = hb.int8_linear(rows, w)
    for lo in (0, m // 2, m - 1000):
        _check_product(got[lo:lo + 1000], x[lo:lo + 1000], rows.scales[lo:lo + 1000], w.values, w.scales, None, None)
    assert hb.device_status() == 0


def test_slices_of_one_buffer():
    """Inputs and outputs that lie side by side in one buffer share no element."""
    import hilberta_b200 as hb
    from hilberta_b200.block_ops import gate_residual_adaln_int8

    buf = _rows(33, 256 + 512 + 64, BF16, seed=1)
    w = hb.quantize_rows(_rows(512, 256, BF16, seed=2))
    want = hb.int8_linear(buf[:, :256].clone(), w)
    before = buf.clone()
    hb.int8_linear(buf[:, :256], w, out=buf[:, 256:768])
    assert torch.equal(buf[:, 256:768], want)
    assert torch.equal(buf[:, :256], before[:, :256]) and torch.equal(buf[:, 768:], before[:, 768:])
    both = _rows(2 * 21, 1024, BF16, seed=3).view(2, 21, 1024)
    x, y = both[..., :512], both[..., 512:]
    shift, scale, gate, *_ = _modulation(2, 512, BF16, seed=4)
    want_x, want_rows = gate_residual_adaln_int8(x.contiguous(), y.contiguous(), gate, shift, scale)
    got, rows = gate_residual_adaln_int8(x, y, gate, shift, scale)
    assert got is x and torch.equal(x, want_x) and torch.equal(rows.values, want_rows.values)
    with pytest.raises(ValueError, match="apart"):
        gate_residual_adaln_int8(x, both[..., 256:768], gate, shift, scale)
    with pytest.raises(ValueError, match="overlap itself"):
        row = both[:1, :1, :512].expand(1, 21, 512)
        gate_residual_adaln_int8(row, both[:1, :, 512:].contiguous(), gate[:1], shift[:1], scale[:1])


def test_int8_linear_row_does_not_depend_on_its_batch():
    import hilberta_b200 as hb

    x, w = _rows(1500, 1024, BF16, seed=1), hb.quantize_rows(_rows(768, 1024, BF16, seed=2))
    want = hb.int8_linear(x, w)
    for lo, hi in ((0, 1), (3, 7), (100, 300), (1100, 1500)):
        assert torch.equal(hb.int8_linear(x[lo:hi], w), want[lo:hi])


def test_int8_linear_streams_graph_and_repeat():
    import hilberta_b200 as hb

    sizes = [(2, 768, 640), (300, 1536, 512), (3000, 512, 1024)]
    cases = [(_rows(m, k, BF16, seed=m), hb.quantize_rows(_rows(n, k, BF16, seed=n))) for m, k, n in sizes]
    want = [hb.int8_linear(x, w, activation="gelu_tanh") for x, w in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        got = []
        for (x, w), s in zip(cases, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(hb.int8_linear(x, w, activation="gelu_tanh"))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [hb.int8_linear(x, w, activation="gelu_tanh") for x, w in cases]
    for x, _ in cases:
        x.mul_(-1.5)
    graph.replay()
    torch.cuda.synchronize()
    for (x, w), o in zip(cases, out):
        assert torch.equal(o, hb.int8_linear(x, w, activation="gelu_tanh"))


@pytest.mark.parametrize("m,k,n", [(5, 512, 384), (40, 1024, 640), (200, 384, 2048), (3000, 256, 1024)])
def test_calls_in_a_row_see_each_other(m, k, n):
    """Producers, quantisation and products back to back, memory reused at once: every
    product sees the values and the weights written just before it."""
    import hilberta_b200 as hb
    from hilberta_b200.block_ops import adaln_int8

    x = _rows(m, k, BF16, seed=1, spread=0.3)
    w = [_rows(n, k, BF16, seed=s, spread=0.0) for s in (2, 3)]
    shift = torch.zeros(1, 256, dtype=BF16, device="cuda")
    want = []
    for i in range(4):
        xi = x * (i + 1) if i % 2 == 0 else x - i
        want.append(hb.int8_linear(hb.quantize_rows(xi), hb.quantize_rows(w[i % 2])))
        torch.cuda.synchronize()
    narrow = x[None, :, :256].contiguous()
    rows = adaln_int8(narrow, shift, shift)
    torch.cuda.synchronize()
    w256 = hb.quantize_rows(w[0][:, :256])
    want_mod = hb.int8_linear(rows, w256)
    torch.cuda.synchronize()
    buf, spare = torch.empty_like(x), torch.empty_like(w[0])
    got, mods = [], []
    for r in range(25):
        for i in range(4):
            torch.mul(x, i + 1, out=buf) if i % 2 == 0 else torch.sub(x, i, out=buf)
            spare.copy_(w[i % 2])
            got.append(hb.int8_linear(buf, hb.quantize_rows(spare)))
        mods.append(hb.int8_linear(adaln_int8(narrow, shift, shift), w256))
    torch.cuda.synchronize()
    for j, g in enumerate(got):
        assert torch.equal(g, want[j % 4]), j
    assert all(torch.equal(g, want_mod) for g in mods)


def _modulation(b, c, dtype, seed):
    return (torch.randn(b, 6 * c, generator=_gen(seed), device="cuda") * 0.5).to(dtype).chunk(6, dim=-1)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("b,s,c", [(1, 1, 256), (2, 77, 768), (3, 130, 3072), (1, 9, 4096)])
def test_adaln_int8(b, s, c, dtype):
    from hilberta_b200.block_ops import adaln_int8, gate_residual, gate_residual_adaln_int8

    x = (_rows(b * s, c, dtype, seed=s, spread=0.5) + 0.5).view(b, s, c)
    y = _rows(b * s, c, dtype, seed=s + 1).view(b, s, c)
    shift, scale, gate, *_ = _modulation(b, c, dtype, seed=c)

    def check(stream, rows):
        f = stream.double()
        h = (f - f.mean(-1, keepdim=True)) / (f.var(-1, correction=0, keepdim=True) + 1e-6).sqrt()
        h = h * (1 + scale.double()[:, None]) + shift.double()[:, None]
        top = h.abs().amax(-1)
        # fp32 mean and variance over C elements and five elementwise steps
        fuzz = 2.0**-19 * (h.abs() + shift.double()[:, None].abs() + top[..., None])
        assert bool(((rows.scales.double() - top / 127).abs() <= top / 127 * 2.0**-17).all())
        off = (rows.values.double() * rows.scales.double()[..., None] - h).abs()
        assert bool((off <= rows.scales.double()[..., None] * 0.5 + fuzz).all())
        assert bool((rows.values.abs().amax(-1) == 127).all())

    rows = adaln_int8(x, shift, scale)
    assert rows.shape == (b, s, c) and rows.dtype == dtype
    check(x, rows)
    apart = torch.empty_like(x)
    before = x.clone()
    got, rows = gate_residual_adaln_int8(x, y, gate, shift, scale, x_out=apart)
    assert got is apart and torch.equal(x, before)
    assert torch.equal(apart, gate_residual(before.clone(), y, gate))
    check(apart, rows)
    got, again = gate_residual_adaln_int8(x, y, gate, shift, scale)
    assert got is x and torch.equal(x, apart) and torch.equal(again.values, rows.values) and torch.equal(again.scales, rows.scales)


def test_adaln_int8_non_finite_rows():
    from hilberta_b200.block_ops import adaln_int8

    x = _rows(12, 512, BF16, seed=1).view(1, 12, 512)
    x[0, 3, 100], x[0, 7, 0] = math.nan, math.inf
    x[0, 5] = 0
    shift, scale, *_ = _modulation(1, 512, BF16, seed=2)
    rows = adaln_int8(x, torch.zeros_like(shift), scale)
    assert rows.scales[0, [3, 7]].isnan().all() and rows.scales[0, 5] == 0
    assert bool((rows.values[0, [3, 5, 7]] == 0).all())
    keep = [i for i in range(12) if i not in (3, 7)]
    assert rows.scales[0, keep].isfinite().all()


def test_modulation_then_products_together():
    """The calls of a block one after the other: modulation, joined Q/K/V product
    into a wider buffer, norms and rotation in place, MLP, joined output projection."""
    import hilberta_b200 as hb
    from hilberta_b200.block_ops import adaln_int8

    b, s, c, heads = 1, 333, 512, 4
    x = _rows(b * s, c, BF16, seed=1, spread=0.3).view(b, s, c)
    shift, scale, *_ = _modulation(b, c, BF16, seed=2)
    wqkv, wup = (hb.quantize_rows((_rows(n, c, BF16, seed=n, spread=0) / math.sqrt(c)).to(BF16)) for n in (3 * c, 4 * c))
    wout = hb.quantize_rows((_rows(c, 5 * c, BF16, seed=3, spread=0) / math.sqrt(5 * c)).to(BF16))
    ones = torch.ones(c // heads, dtype=BF16, device="cuda")
    ang = torch.rand(s, c // heads // 2, generator=_gen(4), device="cuda", dtype=torch.float64) * 6.28
    cos, sin = (f(ang).repeat_interleave(2, 1).float() for f in (torch.cos, torch.sin))
    rows = adaln_int8(x, shift, scale)
    qkv = hb.int8_linear(rows, wqkv).unflatten(-1, (3, heads, c // heads))
    raw = qkv.clone()
    q, k = hb.norm_rope_qk(qkv[:, :, 0], qkv[:, :, 1], weight_q=ones, weight_k=ones, cos=cos, sin=sin,
                           out=(qkv[:, :, 0], qkv[:, :, 1]))
    assert q.data_ptr() == qkv.data_ptr() and torch.equal(qkv[:, :, 2], raw[:, :, 2])
    apart = hb.norm_rope_qk(raw[:, :, 0], raw[:, :, 1], weight_q=ones, weight_k=ones, cos=cos, sin=sin)
    assert torch.equal(apart[0], q) and torch.equal(apart[1], k)
    up = hb.int8_linear(rows, wup, activation="gelu_tanh")
    attn = q.flatten(2)
    out = hb.int8_linear(hb.quantize_rows(attn, joined=up), wout)
    codes, scales = _quantised(torch.cat([attn, up], -1))
    _check_product(out[0], codes[0], scales[0], wout.values, wout.scales, None, None)
    assert hb.device_status() == 0


def test_refusals():
    import hilberta_b200 as hb
    from hilberta_b200.block_ops import adaln_int8

    x = _rows(8, 64, BF16, seed=1)
    w = hb.quantize_rows(_rows(32, 64, BF16, seed=2))
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        hb.quantize_rows(x.float())
    with pytest.raises(ValueError, match="contiguous last"):
        hb.quantize_rows(x.t())
    with pytest.raises(ValueError, match="equally spaced"):
        hb.quantize_rows(_rows(64, 64, BF16, seed=3).view(4, 16, 64)[:, :7])
    with pytest.raises(ValueError, match="leading shape"):
        hb.quantize_rows(x, joined=x[:4])
    with pytest.raises(ValueError, match="disable autograd"):
        hb.quantize_rows(x.clone().requires_grad_())
    with pytest.raises(TypeError, match="Int8Rows"):
        hb.int8_linear(x, x)
    with pytest.raises(ValueError, match="inner size"):
        hb.int8_linear(x[:, :32], w)
    with pytest.raises(ValueError, match="activation"):
        hb.int8_linear(x, w, activation="relu")
    with pytest.raises(ValueError, match="bias"):
        hb.int8_linear(x, w, x[0, :32].float())
    with pytest.raises(ValueError, match="out must be"):
        hb.int8_linear(x, w, out=torch.empty(8, 31, dtype=BF16, device="cuda"))
    with pytest.raises(ValueError, match="overlap itself"):
        hb.int8_linear(x, w, out=torch.empty(1, 32, dtype=BF16, device="cuda").expand(8, 32))
    wide = _rows(8, 96, BF16, seed=4)
    with pytest.raises(ValueError, match="alias"):
        hb.int8_linear(wide[:, :64], w, out=wide[:, 40:72])
    with pytest.raises(ValueError, match="disable autograd"):
        hb.int8_linear(x.clone().requires_grad_(), w)
    values = torch.zeros(4, 72, dtype=torch.int8, device="cuda")
    with pytest.raises(ValueError, match="16-byte aligned"):
        hb.Int8Rows(values, torch.ones(4, device="cuda"), BF16)  # row pitch 72
    with pytest.raises(ValueError, match="one entry per row"):
        hb.Int8Rows(values[:, :64], torch.ones(3, device="cuda"), BF16)
    with pytest.raises(TypeError, match="int8"):
        hb.Int8Rows(values.int(), torch.ones(4, device="cuda"), BF16)
    with pytest.raises(NotImplementedError):
        hb.quantize_rows(torch.zeros(1, 131073, dtype=BF16, device="cuda"))
    m = torch.zeros(1, 128, dtype=BF16, device="cuda")
    with pytest.raises(NotImplementedError, match="multiple of 256"):
        adaln_int8(torch.zeros(1, 8, 128, dtype=BF16, device="cuda"), m, m)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("align", [1, 2, 4, 8])
@pytest.mark.parametrize("k", [16, 1000, 1816, 6008, 15992, 16408])
def test_quantize_rows_by_alignment(k, align, dtype):
    """Rows, parts and lengths that start on 2, 4, 8 or 16 bytes and no more."""
    import hilberta_b200 as hb

    big = _rows(37, k + 5 * align, dtype, seed=k + align)
    pitch = 8 * ((k + 5 * align) // 8 + 1) + align  # elements between rows
    room = torch.full((37 * pitch + 8,), math.nan, dtype=dtype, device="cuda")
    view = room.as_strided((37, k + 5 * align), (pitch, 1), align)
    view.copy_(big)
    for a, b in ((view, None), (view[:, : 3 * align], view[:, 3 * align :]), (view[::2, align:k], view[::2, k:])):
        got = hb.quantize_rows(a, joined=b)
        codes, scales = _quantised(a if b is None else torch.cat([a, b], 1))
        assert torch.equal(got.values, codes) and torch.equal(got.scales, scales)


@pytest.mark.parametrize("b,s,c", [(2, 7001, 256), (1, 9003, 512), (3, 1100, 768), (2, 1501, 1280), (1, 1999, 1536), (2, 801, 2560),
                                   (1, 1201, 2816), (1, 1101, 3328), (3, 602, 3840), (1, 1801, 2048)])
def test_adaln_int8_layouts(b, s, c):
    """Every number of vectors per lane, one warp per row to thirteen, more rows than
    the grid has CTAs, and batch entries that change inside a CTA's rows."""
    from hilberta_b200.block_ops import adaln_int8, gate_residual, gate_residual_adaln_int8

    x = (_rows(b * s, c, BF16, seed=s, spread=0.5) - 0.25).view(b, s, c)
    y = _rows(b * s, c, BF16, seed=s + 1).view(b, s, c)
    shift, scale, gate, *_ = _modulation(b, c, BF16, seed=c)
    stream, joined = gate_residual_adaln_int8(x, y, gate, shift, scale, x_out=torch.empty_like(x))
    assert torch.equal(stream, gate_residual(x.clone(), y, gate))
    for f, rows in ((x.double(), adaln_int8(x, shift, scale)), (stream.double(), joined)):
        h = (f - f.mean(-1, keepdim=True)) / (f.var(-1, correction=0, keepdim=True) + 1e-6).sqrt()
        h = h * (1 + scale.double()[:, None]) + shift.double()[:, None]
        top = h.abs().amax(-1)
        # fp32 mean and variance over C elements and five elementwise steps
        fuzz = 2.0**-19 * (h.abs() + shift.double()[:, None].abs() + top[..., None])
        assert bool(((rows.scales.double() - top / 127).abs() <= top / 127 * 2.0**-17).all())
        off = (rows.values.double() * rows.scales.double()[..., None] - h).abs()
        assert bool((off <= rows.scales.double()[..., None] * 0.5 + fuzz).all())


@pytest.mark.parametrize("rows", [2**31, 2**32 + 5])
def test_more_rows_than_32_bits_count_are_refused(rows):
    import hilberta_b200 as hb

    w = hb.quantize_rows(_rows(1, 1, BF16, seed=1))
    x = torch.ones(1, 1, dtype=BF16, device="cuda").expand(rows, 1)  # rows of one element, all the same
    with pytest.raises(NotImplementedError, match="2.31"):
        hb.quantize_rows(x)
    with pytest.raises(NotImplementedError, match="2.31"):
        hb.int8_linear(x, w)


# Few large tiles and a long K: two CTA pairs share a tile's K (500, 700 tokens), or four.
@pytest.mark.parametrize("dtype,act", [(BF16, None), (FP16, "gelu_tanh")])
@pytest.mark.parametrize("m,n,k", [(500, 3080, 9001), (500, 3079, 9001), (700, 1999, 9000), (1000, 648, 6000),
                                   (260, 1500, 14000), (130, 3330, 14336), (512, 3072, 12288)])
def test_products_with_split_inner_size(m, n, k, dtype, act):
    import hilberta_b200 as hb

    x, w16 = _rows(m, k, dtype, seed=k), _rows(n, k, dtype, seed=n, spread=0.0) * 0.05
    w, bias = hb.quantize_rows(w16), _rows(1, n, dtype, seed=4)[0]
    rows = hb.quantize_rows(x)
    got = hb.int8_linear(rows, w, bias, activation=act)
    _check_product(got, rows.values, rows.scales, w.values, w.scales, bias, act is not None)
    assert torch.equal(got, hb.int8_linear(x, w, bias, activation=act))  # quantised in the call
    few = torch.cat([hb.int8_linear(rows.row_slice(i, i + 60), w, bias, activation=act) for i in range(0, m, 60)])
    assert torch.equal(got, few)  # other kernels, the same integers
    wide = torch.full((m, n + 72), 7.0, dtype=dtype, device="cuda")
    hb.int8_linear(rows, w, bias, activation=act, out=wide[:, 8 : n + 8])
    assert torch.equal(wide[:, 8 : n + 8], got) and bool((wide[:, :8] == 7).all()) and bool((wide[:, n + 8 :] == 7).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = [hb.int8_linear(rows, w, bias, activation=act) for _ in range(3)]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, got) for a in again)
    assert hb.device_status() == 0


# A round of tiles and a few more: the few are shared by two or four pairs each, in a
# second launch that begins while the first ends.
@pytest.mark.parametrize("m,n,k", [(1280, 4096, 9000), (2600, 4093, 8200), (19201, 256, 6200)])
def test_products_with_a_split_last_round(m, n, k):
    import hilberta_b200 as hb

    x, w16 = _rows(m, k, BF16, seed=k), _rows(n, k, BF16, seed=n, spread=0.0) * 0.05
    w, bias = hb.quantize_rows(w16), _rows(1, n, BF16, seed=4)[0]
    rows = hb.quantize_rows(x)
    got = hb.int8_linear(rows, w, bias, activation="gelu_tanh")
    for i in range(0, m, 3000):
        part = rows.row_slice(i, min(m, i + 3000))
        _check_product(got[i : i + 3000], part.values, part.scales, w.values, w.scales, bias, True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = [hb.int8_linear(x, w, bias, activation="gelu_tanh") for _ in range(3)]
        after = hb.quantize_rows(again[2])  # reads all of the product's tiles
    for _ in range(3):
        for a in again:
            a.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, got) for a in again)
    want = hb.quantize_rows(got)
    assert torch.equal(after.values, want.values) and torch.equal(after.scales, want.scales)
    # back to back: codes rewritten by the next call's quantisation as soon as a product ends
    other = x * 0.5
    want = hb.int8_linear(other, w, bias, activation="gelu_tanh")
    for _ in range(10):
        a, b = hb.int8_linear(x, w, bias, activation="gelu_tanh"), hb.int8_linear(other, w, bias, activation="gelu_tanh")
    assert torch.equal(a, got) and torch.equal(b, want) and hb.device_status() == 0


@pytest.mark.parametrize("k", [1024, 1025, 2048, 2049, 3080, 4096, 4100, 5120, 5128, 6144, 6160, 8192, 8193, 10240, 10241, 12288, 12296, 16384, 16385])
def test_quantize_rows_at_every_width_of_a_row(k):
    """The longest row of every number of threads, and one that needs more; more rows than CTAs."""
    import hilberta_b200 as hb

    x = _rows(5003 if k < 5000 else 1201, k, BF16, seed=k)
    got = hb.quantize_rows(x)
    codes, scales = _quantised(x)
    assert torch.equal(got.values, codes) and torch.equal(got.scales, scales)


@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("n,k", [(1, 4096), (4736, 1000), (4737, 515), (9472, 131), (9475, 1001), (20001, 272), (600, 20480)])
def test_one_and_two_tokens(n, k, m):
    """Every number of channels per warp, with channels left over, aligned and odd rows."""
    import hilberta_b200 as hb

    x, w = _rows(m, k, FP16, seed=k), hb.quantize_rows(_rows(n, k, FP16, seed=n % 97, spread=0.0) * 0.05)
    bias, rows = _rows(1, n, FP16, seed=4)[0], hb.quantize_rows(x)
    got = hb.int8_linear(x, w, bias)
    _check_product(got, rows.values, rows.scales, w.values, w.scales, bias, False)
    assert torch.equal(got, hb.int8_linear(rows, w, bias))
    many = hb.int8_linear(torch.cat([x, x, x]), w, bias)  # the tensor-core kernels
    assert torch.equal(many[:m], got)


@pytest.mark.parametrize("m", [3, 4])
@pytest.mark.parametrize("n,k", [(1, 515), (3551, 1001), (3553, 272), (7104, 1000), (7107, 3080), (9000, 131), (20001, 2056), (60, 10240),
                                 (60, 20480)])
def test_three_and_four_tokens(n, k, m):
    """On both sides of the sizes at which the tensor cores take over; every number of
    channels per warp."""
    import hilberta_b200 as hb

    x, w = _rows(m, k, BF16, seed=k), hb.quantize_rows(_rows(n, k, BF16, seed=n % 97, spread=0.0) * 0.05)
    bias, rows = _rows(1, n, BF16, seed=4)[0], hb.quantize_rows(x)
    got = hb.int8_linear(x, w, bias, activation="gelu_tanh")
    _check_product(got, rows.values, rows.scales, w.values, w.scales, bias, True)
    assert torch.equal(got, hb.int8_linear(rows, w, bias, activation="gelu_tanh"))
    assert torch.equal(hb.int8_linear(torch.cat([x, x]), w, bias)[:m], hb.int8_linear(x, w, bias))
    wide = torch.full((m, n + 5), 7.0, dtype=BF16, device="cuda")
    hb.int8_linear(x, w, bias, activation="gelu_tanh", out=wide[:, 2 : n + 2])
    assert torch.equal(wide[:, 2 : n + 2], got) and bool((wide[:, :2] == 7).all()) and bool((wide[:, n + 2 :] == 7).all())


@pytest.mark.parametrize("m,k", [(1, 40960), (2, 20480), (3, 13648), (4, 10240), (2, 131072), (16, 131072), (60, 131072), (200, 131072),
                                 (600, 131072), (1280, 131072)])
@pytest.mark.parametrize("sign", [1, -1])
def test_int8_linear_largest_sums(m, k, sign):
    """Every product 127 * 127 or its negative: sums up to 2114060288, just below 2^31, in
    the dot-product kernel at its longest K and in the tensor-core kernels at theirs."""
    import hilberta_b200 as hb

    n = 144 if k * m < 10**8 else 4096
    x = torch.full((m, k), 127 * sign, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), 127, dtype=torch.int8, device="cuda")
    w[1::2] = -127
    rows = hb.Int8Rows(x, torch.full((m,), 2.0**-16, device="cuda"), BF16)
    weight = hb.Int8Rows(w, torch.ones(n, device="cuda"), BF16)
    want = torch.full((m, n), 16129.0 * k * sign / 2**16, dtype=torch.float64, device="cuda")
    want[:, 1::2] *= -1
    assert torch.equal(hb.int8_linear(rows, weight), want.to(BF16))  # a power of two away from the exact sum
    assert hb.device_status() == 0


def test_modulation_refuses_a_new_stream_that_requires_gradients():
    from hilberta_b200.block_ops import gate_residual_adaln_int8

    x, y = (_rows(9, 256, BF16, seed=s).view(1, 9, 256) for s in (1, 2))
    shift, scale, gate, *_ = _modulation(1, 256, BF16, seed=3)
    out = torch.zeros_like(x, requires_grad=True)
    with pytest.raises(ValueError, match="disable autograd"):
        gate_residual_adaln_int8(x, y, gate, shift, scale, x_out=out)
    with torch.no_grad():
        assert gate_residual_adaln_int8(x, y, gate, shift, scale, x_out=out)[0] is out
