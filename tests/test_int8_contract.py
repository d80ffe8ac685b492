"""Host checks of the 8-bit layer entries and of hb_norm_rope_qk: argument errors
are found before any CUDA call, empty problems return at once.  No GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from hilberta_b200 import _lib, build

    build.build()
    return _lib.lib()


F = ctypes.c_void_p(1 << 20)


def _at(offset):
    return ctypes.c_void_p((1 << 20) + offset)


def test_quantize_rows_checks(lib):
    from hilberta_b200 import _lib

    def call(a=F, a_rs=64, ka=64, b=None, b_rs=0, kb=0, rows=4, codes=F, c_rs=64, scales=F, dtype=1):
        return lib.hb_quantize_rows(a, a_rs, ka, b, b_rs, kb, rows, codes, c_rs, scales, dtype, None)

    for bad in (dict(a=None), dict(codes=None), dict(scales=None), dict(ka=0), dict(kb=-1), dict(rows=-1),
                dict(kb=8), dict(c_rs=48), dict(ka=_lib.HB_INT8_MAX_K, kb=1, b=F)):
        assert call(**bad) == _lib.HB_ERR_ARG, bad
    for bad in (dict(codes=_at(8)), dict(c_rs=72), dict(a=_at(1)), dict(scales=_at(2))):
        assert call(**bad) == _lib.HB_ERR_ALIGN, bad
    assert call(dtype=2) == _lib.HB_ERR_UNSUPPORTED
    assert call(rows=0, a=None, codes=None, scales=None) == _lib.HB_OK


def test_int8_linear_checks(lib):
    from hilberta_b200 import _lib

    def call(x=F, x_rs=64, xs=F, w=F, w_rs=64, ws=F, bias=None, out=F, out_rs=32, M=8, N=32, K=64, act=0, dtype=1):
        return lib.hb_int8_linear(x, x_rs, xs, w, w_rs, ws, bias, out, out_rs, M, N, K, act, dtype, None)

    for bad in (dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(out=None), dict(M=-1), dict(N=-1), dict(K=0),
                dict(K=_lib.HB_INT8_MAX_K + 1, x_rs=1 << 18, w_rs=1 << 18), dict(act=2), dict(x_rs=48), dict(w_rs=48),
                dict(out_rs=31)):
        assert call(**bad) == _lib.HB_ERR_ARG, bad
    for bad in (dict(x=_at(8)), dict(w=_at(4)), dict(x_rs=72), dict(w_rs=72), dict(out=_at(1)), dict(bias=_at(1)), dict(xs=_at(2))):
        assert call(**bad) == _lib.HB_ERR_ALIGN, bad
    assert call(dtype=2) == _lib.HB_ERR_UNSUPPORTED
    assert call(M=0, x=None, out=None) == _lib.HB_OK
    assert call(N=0, w=None, out=None) == _lib.HB_OK
    ws = lib.hb_int8_linear16_workspace_bytes
    assert ws(0, 64) == 0 and ws(1, 0) == 0 and ws(1, 64) == 0  # nothing to do; few tokens stay on chip
    assert ws(100, 70) == 100 * 80 + 400 and ws(8, 131072) == 8 * 131072 + 32

    def call16(x=F, M=100, K=64, w=F, out=F, wsp=F, nbytes=100 * 64 + 400, dtype=1):
        return lib.hb_int8_linear16(x, 64, w, 64, F, None, out, 32, M, 32, K, 0, dtype, wsp, nbytes, None)

    assert call16(x=None) == _lib.HB_ERR_ARG and call16(out=None) == _lib.HB_ERR_ARG and call16(K=0) == _lib.HB_ERR_ARG
    assert call16(x=_at(1)) == _lib.HB_ERR_ALIGN and call16(dtype=3) == _lib.HB_ERR_UNSUPPORTED
    for bad in (dict(wsp=None), dict(nbytes=100 * 64 + 399), dict(wsp=_at(8))):
        assert call16(**bad) == _lib.HB_ERR_WORKSPACE, bad
    assert call16(M=0, x=None, wsp=None) == _lib.HB_OK
    assert lib.hb_int8_status(0, None, None) == _lib.HB_ERR_ARG


def test_adaln_residual_int8_checks(lib):
    from hilberta_b200 import _lib

    def call(x=F, rs=512, y=F, gate=F, shift=F, scale=F, mod=512, xo=F, codes=F, c_rs=512, scales=F, rows=4, per=4, C=512,
             eps=1e-6, dtype=1):
        return lib.hb_adaln_residual_int8(x, rs, y, rs, gate, shift, scale, mod, xo, rs, codes, c_rs, scales, rows, per, C,
                                          eps, dtype, None)

    for bad in (dict(x=None), dict(codes=None), dict(scales=None), dict(shift=None), dict(scale=None), dict(gate=None),
                dict(xo=None), dict(rows=-1), dict(per=0), dict(eps=-1.0), dict(c_rs=256)):
        assert call(**bad) == _lib.HB_ERR_ARG, bad
    for bad in (dict(C=128, c_rs=128), dict(C=4352, c_rs=4352), dict(dtype=2)):
        assert call(**bad) == _lib.HB_ERR_UNSUPPORTED, bad
    for bad in (dict(x=_at(8)), dict(codes=_at(8)), dict(rs=516), dict(c_rs=520), dict(mod=4), dict(scales=_at(2))):
        assert call(**bad) == _lib.HB_ERR_ALIGN, bad
    assert call(rows=0) == _lib.HB_OK
    assert call(rows=0, y=None, gate=None, xo=None) == _lib.HB_OK


def test_norm_rope_qk_checks(lib):
    from hilberta_b200 import _lib

    def call(q=F, k=F, qo=F, ko=F, B=1, S=4, T=0, Hq=2, Hk=1, D=64, wq=F, wtq=None, cos=F, sn=128, eps=1e-6, dtype=1):
        strides = (ctypes.c_int64 * 12)(*[4 * sn, sn, 64] * 4)
        return lib.hb_norm_rope_qk(q, k, qo, ko, strides, B, S, T, Hq, Hk, D, wq, F, wtq, wtq, eps, cos, F, dtype, None)

    for bad in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(B=-1), dict(S=-1), dict(T=5), dict(T=-1),
                dict(T=2), dict(Hq=0), dict(Hk=0), dict(wq=None), dict(cos=None), dict(eps=-1.0)):
        assert call(**bad) == _lib.HB_ERR_ARG, bad
    for bad in (dict(q=_at(8)), dict(ko=_at(4)), dict(wq=_at(8)), dict(cos=_at(8)), dict(sn=132), dict(T=2, wtq=_at(8))):
        assert call(**bad) == _lib.HB_ERR_ALIGN, bad
    for bad in (dict(D=96), dict(D=16), dict(dtype=2)):
        assert call(**bad) == _lib.HB_ERR_UNSUPPORTED, bad
    assert call(B=0) == _lib.HB_OK and call(S=0, q=None) == _lib.HB_OK


def test_python_entries_want_cuda_tensors():
    import hilberta_b200 as hb

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        hb.quantize_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        hb.Int8Rows(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4), torch.bfloat16)
    with pytest.raises(TypeError, match="Int8Rows"):
        hb.int8_linear(x, x)
    h = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        hb.norm_rope_qk(h, h, weight_q=x[0], weight_k=x[0], cos=x.float(), sin=x.float())


def test_row_strides():
    from hilberta_b200.int8 import _row_stride

    t = torch.empty(4, 6, 32)
    assert _row_stride(t) == 32 and _row_stride(t[:, :, :16]) == 32 and _row_stride(t[0]) == 32
    assert _row_stride(t[:, :5]) is None and _row_stride(t[::2]) is None
    assert _row_stride(t[:1, :5]) == 32 and _row_stride(t[:, :1]) == 192 and _row_stride(t.view(2, 2, 6, 32)) == 32
    assert _row_stride(t[:1, :1]) == 32 and _row_stride(t[:, ::2]) == 64


def test_wait_limit_checks(lib):
    from hilberta_b200 import _lib

    assert lib.hb_int8_set_wait_limit(-1) == _lib.HB_ERR_ARG
    assert lib.hb_int8_set_wait_limit(0) == _lib.HB_OK and lib.hb_int8_set_wait_limit(2000) == _lib.HB_OK
