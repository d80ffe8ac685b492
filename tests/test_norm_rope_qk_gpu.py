"""hb_norm_rope_qk against its formula in 64 bits.

fp32 inside, one rounding at the end: eps/2 of the result, and the fp32 steps.
The sum of D squares is taken in 8 + log2(D/8) additions (2^-24 each), the
reciprocal root is within 2^-22, weight, scale and rotation add five roundings:
together below 2^-20 of each of the two terms of a rotated element.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _case(b, s, hq, hk, d, dtype, seed=1, text=0):
    g = _gen(seed)
    q, k = ((3 * torch.randn(b, s, h, d, generator=g, device="cuda")).to(dtype) for h in (hq, hk))
    w = [(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype) for _ in range(4)]
    ang = torch.rand(s, d // 2, generator=g, device="cuda", dtype=torch.float64) * 100
    cos, sin = (f(ang).repeat_interleave(2, 1).float() for f in (torch.cos, torch.sin))
    kw = dict(weight_q=w[0], weight_k=w[1], cos=cos, sin=sin)
    if text:
        kw |= dict(text_tokens=text, weight_txt_q=w[2], weight_txt_k=w[3])
    return q, k, kw


def _check(got, x, w, w_txt, kw, eps=1e-6):
    f = x.double()
    rows = w.double().expand(f.shape[1], -1).clone()
    if w_txt is not None:
        rows[:kw["text_tokens"]] = w_txt.double()
    z = f / (f.square().mean(-1, keepdim=True) + eps).sqrt() * rows[:, None]
    a, c = z[..., 0::2], z[..., 1::2]
    cos, sin = kw["cos"].double()[:, None], kw["sin"].double()[:, None]
    terms = [(a * cos[..., 0::2], -c * sin[..., 0::2]), (c * cos[..., 1::2], a * sin[..., 1::2])]
    half = torch.finfo(x.dtype).eps / 2
    tiny = 2.0**-25 if x.dtype == FP16 else 0.0
    for i, (u, v) in enumerate(terms):
        ref = u + v
        bound = ref.abs() * half + 2.0**-20 * (u.abs() + v.abs()) + tiny
        err = (got[..., i::2].double() - ref).abs()
        assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("b,s,hq,hk,text", [(1, 1, 1, 1, 0), (1, 1, 24, 24, 1), (3, 7, 5, 1, 2), (2, 513, 20, 4, 0),
                                            (1, 2000, 24, 24, 512), (4, 33, 3, 7, 33)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_against_formula(b, s, hq, hk, text, d, dtype):
    import hilberta_b200 as hb

    q, k, kw = _case(b, s, hq, hk, d, dtype, seed=s + d, text=text)
    before = q.clone(), k.clone()
    qo, ko = hb.norm_rope_qk(q, k, **kw)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    _check(qo, q, kw["weight_q"], kw.get("weight_txt_q"), kw)
    _check(ko, k, kw["weight_k"], kw.get("weight_txt_k"), kw)


@pytest.mark.parametrize("text", [0, 5])
def test_in_place_in_a_joined_projection(text):
    """Query and key slices of one [B, S, (2 Hq' ...)] buffer, in place: the value part and the result are what
    separate tensors give; views over heads-first storage too."""
    import hilberta_b200 as hb

    b, s, h, d = 2, 77, 6, 64
    q, k, kw = _case(b, s, h, h, d, BF16, text=text)
    want = hb.norm_rope_qk(q, k, **kw)
    buf = torch.full((b, s, 3, h, d), 9.0, dtype=BF16, device="cuda")
    buf[:, :, 0], buf[:, :, 1] = q, k
    views = (buf[:, :, 0], buf[:, :, 1])
    got = hb.norm_rope_qk(*views, out=views, **kw)
    assert got[0].data_ptr() == buf.data_ptr()
    assert torch.equal(buf[:, :, 0], want[0]) and torch.equal(buf[:, :, 1], want[1]) and bool((buf[:, :, 2] == 9.0).all())
    qt, kt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k))  # [B, H, S, D] storage
    got = hb.norm_rope_qk(qt, kt, out=(qt, kt), **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_zero_and_non_finite_rows_and_empty():
    import hilberta_b200 as hb

    q, k, kw = _case(1, 9, 4, 2, 128, BF16)
    q[0, 2, 1] = 0
    q[0, 3, 0, 5] = math.inf
    k[0, 4, 1, 7] = math.nan
    qo, ko = hb.norm_rope_qk(q, k, **kw)
    assert bool((qo[0, 2, 1] == 0).all()) and ko[0, 4, 1].isnan().all() and qo[0, 3, 0].isnan().any()
    clean = torch.ones(9, 4, dtype=torch.bool)
    clean[3, 0] = False
    assert qo[0][clean].isfinite().all()
    kw["cos"], kw["sin"] = kw["cos"][:0], kw["sin"][:0]
    qo, ko = hb.norm_rope_qk(q[:, :0], k[:, :0], **kw)
    assert qo.shape == (1, 0, 4, 128) and ko.shape == (1, 0, 2, 128)


def test_graph_and_other_stream():
    import hilberta_b200 as hb

    q, k, kw = _case(1, 300, 24, 24, 128, BF16, text=20)
    want = hb.norm_rope_qk(q, k, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = hb.norm_rope_qk(q, k, **kw)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = hb.norm_rope_qk(q, k, **kw)
    q.mul_(-2), k.add_(1)
    graph.replay()
    torch.cuda.synchronize()
    want = hb.norm_rope_qk(q, k, **kw)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    import hilberta_b200 as hb

    q, k, kw = _case(2, 8, 4, 2, 64, BF16)
    call = lambda q=q, k=k, **c: hb.norm_rope_qk(q, k, **{**kw, **c})  # noqa: E731
    with pytest.raises(ValueError, match="agree"):
        call(k=k[:1])
    with pytest.raises(ValueError, match="agree"):
        call(k=k.half())
    with pytest.raises(TypeError):
        call(q=q.float(), k=k.float())
    with pytest.raises(ValueError, match="text_tokens"):
        call(text_tokens=9)
    with pytest.raises(ValueError, match="weight_txt"):
        call(text_tokens=2)
    with pytest.raises(ValueError, match="norm weights"):
        call(weight_q=kw["weight_q"].float())
    with pytest.raises(ValueError, match="cos/sin"):
        call(cos=kw["cos"][:4])
    with pytest.raises(ValueError, match="eps"):
        call(eps=-1.0)
    with pytest.raises(ValueError, match="disable autograd"):
        call(q=q.clone().requires_grad_())
    with pytest.raises(ValueError, match="in place or must not overlap"):
        call(out=(q[:, :, [0, 1, 2, 3]].clone(), k)) and call(out=(q, q[:, :, 1:3]))
    with pytest.raises(ValueError, match="in place or must not overlap"):
        wide = torch.zeros(2, 8, 5, 64, dtype=BF16, device="cuda")
        call(q=wide[:, :, :4], out=(wide[:, :, 1:], k.clone()))
    with pytest.raises(ValueError, match="overlap itself"):
        call(out=(q, k[:, :, :1].expand(2, 8, 2, 64)))
    with pytest.raises(ValueError, match="aligned"):
        odd = torch.zeros(2, 8, 4, 68, dtype=BF16, device="cuda")[..., 4:]
        call(q=odd)
    with pytest.raises(NotImplementedError):
        x = torch.zeros(1, 1, 1, 48, dtype=BF16, device="cuda")
        t = torch.zeros(1, 48, device="cuda")
        hb.norm_rope_qk(x, x.clone(), weight_q=x[0, 0, 0], weight_k=x[0, 0, 0], cos=t, sin=t)
