"""The four query/key norms of an 8-bit attention module each use their own eps."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

EPS = dict(norm_q=0.5, norm_k=1e-6, norm_added_q=0.5, norm_added_k=3.0)


def _plain(q, k, *, weight_q, weight_k, cos, sin, text_tokens=0, weight_txt_q=None, weight_txt_k=None, eps=1e-6, out=None):
    """The formula in 64 bits (in place of the kernel)."""
    got = []
    for x, w, w_txt in ((q, weight_q, weight_txt_q), (k, weight_k, weight_txt_k)):
        z = x.double() * (x.double().square().mean(-1, keepdim=True) + eps).rsqrt()
        rows = w.double().expand(x.shape[1], 1, -1).clone()
        if text_tokens:
            rows[:text_tokens] = w_txt.double()
        z = z * rows
        turned = torch.stack([-z[..., 1::2], z[..., 0::2]], -1).flatten(-2)
        got.append((z * cos.double()[:, None] + turned * sin.double()[:, None]).to(x.dtype))
    if out is None:
        return tuple(got)
    for o, g in zip(out, got):
        o.copy_(g)
    return out


def _module(T, n, heads=2, d=32):
    """An 8-bit attention module on the CPU whose projections copy ready rows."""
    from hilberta_b200.flux_int8 import Int8JointAttention

    g = torch.Generator().manual_seed(T + n)

    class Rows(torch.nn.Module):
        def __init__(self, tokens):
            super().__init__()
            self.values = torch.empty(3 * heads * d, 0)
            self.rows = torch.randn(2, tokens, 3 * heads * d, generator=g).to(torch.bfloat16)

        def forward(self, x, out):
            out.copy_(self.rows)

    attn = Int8JointAttention.__new__(Int8JointAttention)
    torch.nn.Module.__init__(attn)
    attn.heads, attn.to_qkv, attn.add_qkv = heads, Rows(n), Rows(T)
    for name in EPS:
        setattr(attn, name, SimpleNamespace(weight=torch.randn(d, generator=g).to(torch.bfloat16), eps=1e-6))
    cos, sin = torch.randn(T + n, d, generator=g), torch.randn(T + n, d, generator=g)
    return attn, torch.zeros(2, n, 8, dtype=torch.bfloat16), torch.zeros(2, T, 8, dtype=torch.bfloat16) if T else None, (cos, sin)


@pytest.mark.parametrize("T,n", [(5, 7), (0, 6), (3, 1)])
@pytest.mark.parametrize("names", [(), ("norm_k",), tuple(EPS)])
def test_each_norm_by_its_own_eps(T, n, names, monkeypatch):
    from hilberta_b200 import flux_int8

    monkeypatch.setattr(flux_int8, "norm_rope_qk", _plain)
    attn, image, text, rot = _module(T, n)
    for name in names:
        getattr(attn, name).eps = EPS[name]
    got = [x.transpose(1, 2) for x in attn.joint_qkv(image, text, rot)]
    rows = torch.cat([attn.add_qkv.rows, attn.to_qkv.rows], 1) if T else attn.to_qkv.rows
    raw = rows.view(2, T + n, 3, 2, 32).unbind(2)
    for lo, hi, q_norm, k_norm in ((0, T, attn.norm_added_q, attn.norm_added_k), (T, T + n, attn.norm_q, attn.norm_k)):
        for i, norm in enumerate((q_norm, k_norm)):
            part = raw[i][:, lo:hi]
            want = _plain(part, part, weight_q=norm.weight, weight_k=norm.weight, cos=rot[0][lo:hi], sin=rot[1][lo:hi], eps=norm.eps)
            assert torch.equal(got[i][:, lo:hi], want[0]), (i, lo)
    assert torch.equal(got[2], raw[2])


@pytest.mark.gpu
def test_each_norm_by_its_own_eps_on_the_device():
    import hilberta_b200 as hb
    from hilberta_b200.flux_int8 import quantize_flux_model
    from hilberta_b200.flux_model import FluxTransformer

    torch.manual_seed(0)
    model = quantize_flux_model(FluxTransformer(num_double=1, num_single=1, dim=256, heads=2, text_dim=64, pooled_dim=32, device="cuda"))
    attn = model.transformer_blocks[0].attn
    T, n = 9, 40
    image, text = (torch.randn(2, t, 256, device="cuda").to(torch.bfloat16) for t in (n, T))
    cos, sin = torch.randn(T + n, 128, device="cuda"), torch.randn(T + n, 128, device="cuda")
    with torch.inference_mode():
        rows = torch.cat([attn.add_qkv(text), attn.to_qkv(image)], 1)
        raw = rows.view(2, T + n, 3, 2, 128).unbind(2)
        for eps in ((1e-6,) * 4, tuple(EPS.values())):
            for name, e in zip(EPS, eps):
                getattr(attn, name).eps = e
            got = [x.transpose(1, 2) for x in attn.joint_qkv(image, text, (cos, sin))]
            for lo, hi, norms in ((0, T, (attn.norm_added_q, attn.norm_added_k)), (T, T + n, (attn.norm_q, attn.norm_k))):
                for i, norm in enumerate(norms):
                    part = raw[i][:, lo:hi]
                    want = hb.norm_rope_qk(part, part, weight_q=norm.weight, weight_k=norm.weight, cos=cos[lo:hi], sin=sin[lo:hi],
                                           eps=norm.eps)
                    assert torch.equal(got[i][:, lo:hi], want[0])
            assert torch.equal(got[2], raw[2])
