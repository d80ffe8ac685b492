"""Q/K/V preparation in front of the attention (``hb_norm_rope_pack``).

The FLUX processor (hilberta/flux_adapter.py:280-298) turns the six projections
of a double-stream block into the attention inputs:

* split each projection into heads (``unflatten(-1, (heads, -1))``);
* RMS-normalise query and key rows over the head dimension (``norm_q`` /
  ``norm_k`` for the image stream, ``norm_added_q`` / ``norm_added_k`` for the
  text stream; learned weight, eps 1e-6 in FLUX);
* concatenate text tokens first, image tokens after;
* rotate query and key by the rotary embedding (``apply_rotary_emb`` with real
  cos/sin of shape [S, D]);
* hand ``transpose(1, 2)`` views ([B, H, S, D] of [B, S, H, D] storage) to the
  attention.

``prepare_qkv`` does all of it with one pass over HBM per tensor and returns
those views, ready for ``paired_attention``.  ``image_rows`` optionally writes
image token i to token ``T + image_rows[i]`` (for instance the plan's inverse
order, giving the physical layout the plain kernel reads).  No CPU path.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from .int8 import _overlaps_itself, _span


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return 1
    if t.dtype == torch.float16:
        return 0
    raise TypeError("16-bit (bf16/fp16) projections required")


def norm_rope_pack(txt, img, *, heads, weight_txt=None, weight_img=None, eps=1e-6, cos=None, sin=None,
                   image_rows=None, out=None):
    """One of Q/K/V: ``txt`` [B, T, heads*D] and ``img`` [B, n, heads*D] (D
    contiguous, 16-bit) -> [B, T+n, heads, D] (``out`` if given).  Weights [D]
    in the inputs' dtype (both or neither); cos/sin fp32 [T+n, D] by output
    token (both or neither)."""
    ref = img if img is not None else txt
    if ref is None or not ref.is_cuda:
        raise ValueError("CUDA projections required")
    B = ref.shape[0]
    HD = ref.shape[-1]
    if HD % heads:
        raise ValueError("projection width must split into heads")
    D = HD // heads
    T = 0 if txt is None else txt.shape[1]
    n = 0 if img is None else img.shape[1]
    for x in (txt, img):
        if x is not None and (x.ndim != 3 or x.shape[0] != B or x.shape[2] != HD or x.stride(-1) != 1
                              or x.dtype != ref.dtype or x.device != ref.device):
            raise ValueError("txt/img must be [B, tokens, heads*D] with contiguous last dim, same dtype/device")
    if (weight_txt is None) != (weight_img is None):
        raise ValueError("give both stream weights or neither")
    for w in (weight_txt, weight_img):
        if w is not None and (w.shape != (D,) or w.dtype != ref.dtype or w.device != ref.device or not w.is_contiguous()):
            raise ValueError("norm weights must be contiguous [D] in the projections' dtype")
    if (cos is None) != (sin is None):
        raise ValueError("give both cos and sin or neither")
    for c in (cos, sin):
        if c is not None and (c.shape != (T + n, D) or c.dtype != torch.float32 or c.device != ref.device
                              or not c.is_contiguous()):
            raise ValueError("cos/sin must be contiguous fp32 [T+n, D] on the projections' device")
    if image_rows is not None and (image_rows.shape != (n,) or image_rows.dtype != torch.int32
                                   or image_rows.device != ref.device or not image_rows.is_contiguous()):
        raise ValueError("image_rows must be a contiguous int32 [n] tensor on the projections' device")
    if out is None:
        out = torch.empty((B, T + n, heads, D), dtype=ref.dtype, device=ref.device)
    elif out.shape != (B, T + n, heads, D) or out.dtype != ref.dtype or out.stride(-1) != 1:
        raise ValueError("out must be [B, T+n, heads, D] with contiguous D")
    status = None
    rc = _lib.lib().hb_norm_rope_pack(
        _lib.ptr(txt), 0 if txt is None else txt.stride(0), 0 if txt is None else txt.stride(1),
        _lib.ptr(img), 0 if img is None else img.stride(0), 0 if img is None else img.stride(1),
        B, T, n, heads, D, _lib.ptr(weight_txt), _lib.ptr(weight_img), float(eps), _lib.ptr(cos), _lib.ptr(sin),
        _lib.ptr(image_rows), _lib.ptr(out), out.stride(0), out.stride(1), out.stride(2), _dtype_code(ref), status,
        ctypes.c_void_p(torch.cuda.current_stream(ref.device).cuda_stream),
    )
    if rc == _lib.HB_ERR_ALIGN:
        raise ValueError("hb_norm_rope_pack needs 16-byte aligned rows (strides multiples of 8 elements)")
    if rc == _lib.HB_ERR_UNSUPPORTED:
        raise NotImplementedError("hb_norm_rope_pack supports D 64 or 128, fp16/bf16")
    _lib.check(rc, "hb_norm_rope_pack")
    return out


def prepare_qkv(q_txt, k_txt, v_txt, q_img, k_img, v_img, *, heads, norm_q, norm_k, norm_added_q, norm_added_k,
                rotary=None, eps=1e-6, image_rows=None):
    """The processor's Q/K/V for the attention: [B, H, S, D] views of [B, S, H, D]
    storage, text tokens first.  norm_* are the [D] RMSNorm weights; rotary is
    (cos, sin), fp32 [S, D] by output token, or None."""
    cos, sin = (None, None) if rotary is None else rotary
    q = norm_rope_pack(q_txt, q_img, heads=heads, weight_txt=norm_added_q, weight_img=norm_q, eps=eps, cos=cos,
                       sin=sin, image_rows=image_rows)
    k = norm_rope_pack(k_txt, k_img, heads=heads, weight_txt=norm_added_k, weight_img=norm_k, eps=eps, cos=cos,
                       sin=sin, image_rows=image_rows)
    v = norm_rope_pack(v_txt, v_img, heads=heads, image_rows=image_rows)
    return q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)


_STRIDES = struct.Struct("12q")


def norm_rope_qk(q, k, *, weight_q, weight_k, cos, sin, text_tokens=0, weight_txt_q=None, weight_txt_k=None, eps=1e-6,
                 out=None):
    """RMSNorm over the head dimension and rotary embedding of query and key heads,
    both in one launch (``hb_norm_rope_qk``).

    ``q`` [B, S, Hq, D] and ``k`` [B, S, Hk, D] (Hk may differ: shared key heads),
    16-bit, D 32/64/128/256 contiguous, any 16-byte aligned outer strides: e.g. the
    query and key slices of one joined projection.  Weights [D] in the same type;
    the first ``text_tokens`` tokens use ``weight_txt_q`` / ``weight_txt_k``.
    ``cos``/``sin`` fp32 [S, D] by token, pairs (2i, 2i+1).  Arithmetic is fp32 with
    one rounding at the end (``norm_rope_pack`` keeps the rounding of the separate
    ops it replaces).  ``out`` is a pair of tensors like q and k, ``(q, k)`` itself
    for in place; by default new contiguous ones.  Returns the pair."""
    if q.ndim != 4 or k.ndim != 4 or not q.is_cuda or q.stride()[3] != 1 or k.stride()[3] != 1:
        raise ValueError("q and k must be CUDA tensors [B, S, heads, D] with contiguous D")
    kind, dev = q.dtype, q.device
    dtype = _dtype_code(q)
    B, S, Hq, D = q.shape
    Hk = k.shape[2]
    if k.shape != (B, S, Hk, D) or k.dtype != kind or k.device != dev:
        raise ValueError("q and k must agree in batch, tokens, D, dtype and device")
    if Hq < 1 or Hk < 1:
        raise ValueError("at least one query and one key head required")
    T = int(text_tokens)
    if not 0 <= T <= S:
        raise ValueError("text_tokens must lie within the tokens")
    if T > 0 and (weight_txt_q is None or weight_txt_k is None):
        raise ValueError("text tokens need weight_txt_q and weight_txt_k")
    weights = (weight_q, weight_k) if weight_txt_q is None and weight_txt_k is None else (weight_q, weight_k, weight_txt_q,
                                                                                        weight_txt_k)
    for w in weights:
        if w is not None and (w.shape != (D,) or w.dtype != kind or w.device != dev or not w.is_contiguous()):
            raise ValueError("norm weights must be contiguous [D] in the heads' dtype")
    for c in (cos, sin):
        if c is None or c.shape != (S, D) or c.dtype != torch.float32 or c.device != dev or not c.is_contiguous():
            raise ValueError("cos/sin must be contiguous fp32 [S, D] on the heads' device")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if torch.is_grad_enabled():
        for t in (q, k, cos, sin, *weights):
            if t is not None and t.requires_grad:
                raise ValueError("Inference only; disable autograd")
    if out is None:
        q_out, k_out = q.new_empty(B, S, Hq, D), k.new_empty(B, S, Hk, D)
    else:
        _check_qk_out(q, k, out, [t for t in (cos, sin, *weights) if t is not None])
        q_out, k_out = out
    strides = _STRIDES.pack(*q.stride()[:3], *k.stride()[:3], *q_out.stride()[:3], *k_out.stride()[:3])
    with _lib.on_device(dev) as stream:
        rc = _lib.lib().hb_norm_rope_qk(
            q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), strides, B, S, T, Hq, Hk, D,
            weight_q.data_ptr(), weight_k.data_ptr(), None if weight_txt_q is None else weight_txt_q.data_ptr(),
            None if weight_txt_k is None else weight_txt_k.data_ptr(), eps, cos.data_ptr(), sin.data_ptr(), dtype,
            stream)
    if rc == _lib.HB_ERR_ALIGN:
        raise ValueError("hb_norm_rope_qk needs 16-byte aligned rows (strides multiples of 8 elements)")
    if rc == _lib.HB_ERR_UNSUPPORTED:
        raise NotImplementedError("hb_norm_rope_qk supports D 32, 64, 128 or 256, fp16/bf16")
    _lib.check(rc, "hb_norm_rope_qk")
    return q_out, k_out


def _check_qk_out(q, k, out, others):
    """Outputs: like q and k, each either its input in place or apart from everything read.
    ``others`` are contiguous."""
    q_out, k_out = out
    in_place = q_out is q and k_out is k
    for name, x, o in (("q", q, q_out), ("k", k, k_out)):
        if not in_place:
            if o.shape != x.shape or o.dtype != x.dtype or o.device != x.device or o.stride(-1) != 1:
                raise ValueError(f"the output of {name} must match its shape, dtype and device with contiguous D")
            if torch.is_grad_enabled() and o.requires_grad:
                raise ValueError("Inference output cannot require gradients")
        if _overlaps_itself(o):
            raise ValueError(f"the output of {name} must not overlap itself")
    same = [in_place or o.data_ptr() == x.data_ptr() and o.stride() == x.stride() for x, o in ((q, q_out), (k, k_out))]
    if all(same) and _interleaved(q, k):
        begin, end = _rows_span(q)
        first, last = _rows_span(k)
        begin, end = min(begin, first), max(end, last)
        for t in others:
            first = t.data_ptr()
            if first < end and (first >= begin or first + t.numel() * t.element_size() > begin):
                raise ValueError("norm weights and cos/sin must not overlap the outputs")
        return
    for o, over, own, rest in ((q_out, same[0], q, (k, k_out)), (k_out, same[1], k, (q, q_out))):
        begin, end = _span(o)
        for t in (*rest, *others) if over else (own, *rest, *others):
            first, last = _span(t)
            if begin < last and first < end and not (t.dtype == o.dtype and _interleaved(o, t)):
                raise ValueError("outputs must be their inputs in place or must not overlap any input")


def _rows_span(t):
    """``_span`` of a nonempty 16-bit [B, S, heads, D] with contiguous D."""
    B, S, H, D = t.shape
    entry, token, head, _ = t.stride()
    first = t.data_ptr()
    return first, first + 2 * ((B - 1) * entry + (S - 1) * token + (H - 1) * head + D)


def _interleaved(a, b):
    """a and b are slices of equally strided rows, side by side within the token stride
    (as the query and key parts of one joined projection) or the batch stride (as parts
    of [B, 3, S, heads, D]), sharing no element."""
    if a.ndim != 4 or b.ndim != 4 or a.stride()[:2] != b.stride()[:2]:
        return False
    entry, token = a.stride()[:2]
    many, tokens = max(a.shape[0], b.shape[0]) > 1, max(a.shape[1], b.shape[1])
    width = lambda t: (t.shape[2] - 1) * t.stride(2) + t.shape[3]  # noqa: E731
    wide, other = width(a), width(b)
    apart = (b.data_ptr() - a.data_ptr()) // a.element_size()
    # Batch entries that are no whole number of tokens apart: only a row's own
    # neighbourhood is known, not where it meets the rows of another entry.
    if token > 0 and (not many or entry >= tokens * token and (entry % token == 0 or abs(apart) < token)):
        if apart % token >= wide and apart % token + other <= token:
            return True
    if not many or entry <= 0:
        return False
    wide, other = wide + (a.shape[1] - 1) * token, other + (b.shape[1] - 1) * token
    return apart % entry >= wide and apart % entry + other <= entry
