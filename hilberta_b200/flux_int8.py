"""The FLUX.1-architecture transformer with 8-bit weights and activations.

``quantize_flux_model(model)`` rewrites a ``flux_model.FluxTransformer`` in place:

* every projection of the blocks (Q/K/V, attention outputs, MLPs, adaLN
  modulation) becomes an ``Int8Linear``: weights quantised once per output
  channel, tokens per call and token, products summed exactly in integers;
* Q, K and V of a stream are one product, written where the attention reads them:
  text and image tokens go to their places in one ``[B, S, 3, H, D]`` buffer, whose
  query and key parts are normalised and rotated in place by one
  ``norm_rope_qk``, while the value part is not touched again;
* the modulation in front of a projection quantises its output in the same pass
  (``adaln_int8`` / ``gate_residual_adaln_int8``), and the single-stream output
  projection quantises [attention | MLP] without concatenating them.

Embedders, the output layer, norms, residual stream and attention stay in 16
bits.  The model keeps its forward signature and processors, so
``persistent_flux_attention`` and ``sample_flux_persistent`` apply unchanged.
The reference has no counterpart (its adapter reports "weights_modified: False").
"""

from __future__ import annotations

import functools

import torch

from .block_ops import NativeBlockOps, adaln_int8, gate_residual_adaln_int8
from .flux_model import FluxTransformer
from .int8 import Int8Linear, int8_linear, quantize_rows
from .prep import norm_rope_qk


class Int8BlockOps(NativeBlockOps):
    """``NativeBlockOps`` whose modulated tokens are ``Int8Rows``."""

    @staticmethod
    def modulate(x, shift, scale):
        return adaln_int8(x, shift, scale)

    @staticmethod
    def gate_add_modulate(x, y, gate, shift, scale):
        return gate_residual_adaln_int8(x, y, gate, shift, scale)

    @staticmethod
    def linear_gelu(x, weight, bias):
        return int8_linear(x, weight, bias, activation="gelu_tanh")


class Int8JoinedLinear(torch.nn.Module):
    """``flux_model.JoinedLinear`` in 8 bits: [attention | MLP] is quantised as one
    row per token (one scale) and multiplied once."""

    def __init__(self, joined):
        super().__init__()
        self.layer = Int8Linear(joined)

    def forward(self, a, m, ops):
        return self.layer(quantize_rows(a, joined=m))


class Int8JointAttention(torch.nn.Module):
    """``flux_model.JointAttention`` in 8 bits.  Processors take q, k and v from
    ``joint_qkv``; the separate projections (``to_q`` and so on) are slices of the
    joined ones."""

    def __init__(self, attn):
        super().__init__()
        self.heads, self.added_kv_proj_dim = attn.heads, attn.added_kv_proj_dim
        self.to_qkv = Int8Linear.joined([attn.to_q, attn.to_k, attn.to_v])
        self.norm_q, self.norm_k = attn.norm_q, attn.norm_k
        if attn.added_kv_proj_dim is not None:
            self.add_qkv = Int8Linear.joined([attn.add_q_proj, attn.add_k_proj, attn.add_v_proj])
            self.norm_added_q, self.norm_added_k = attn.norm_added_q, attn.norm_added_k
            self.to_out = torch.nn.ModuleList([Int8Linear(attn.to_out[0]), attn.to_out[1]])
            self.to_add_out = Int8Linear(attn.to_add_out)
        self.processor = attn.processor

    def set_processor(self, processor):
        self.processor = processor

    def forward(self, hidden_states, encoder_hidden_states=None, image_rotary_emb=None):
        return self.processor(self, hidden_states, encoder_hidden_states, image_rotary_emb=image_rotary_emb)

    def _part(self, layer, i):
        inner = layer.values.shape[0] // 3
        return layer.outputs(i * inner, (i + 1) * inner)

    to_q = property(lambda self: self._part(self.to_qkv, 0))
    to_k = property(lambda self: self._part(self.to_qkv, 1))
    to_v = property(lambda self: self._part(self.to_qkv, 2))
    add_q_proj = property(lambda self: self._part(self.add_qkv, 0))
    add_k_proj = property(lambda self: self._part(self.add_qkv, 1))
    add_v_proj = property(lambda self: self._part(self.add_qkv, 2))

    def joint_qkv(self, hidden_states, encoder_hidden_states, image_rotary_emb):
        """(q, k, v) as [B, H, S, D] views of one [B, S, 3, H, D] buffer, text tokens
        first, q and k normalised and rotated."""
        if image_rotary_emb is None:
            raise ValueError("8-bit attention needs the rotary embedding")
        B, n = hidden_states.shape[:2]
        T = 0 if encoder_hidden_states is None else encoder_hidden_states.shape[1]
        width = self.to_qkv.values.shape[0]
        buf = torch.empty((B, T + n, width), dtype=hidden_states.dtype, device=hidden_states.device)
        self.to_qkv(hidden_states, out=buf[:, T:])
        text, norms = {}, [(self.norm_q, self.norm_k)]
        if T:
            self.add_qkv(encoder_hidden_states, out=buf[:, :T])
            text = dict(text_tokens=T, weight_txt_q=self.norm_added_q.weight, weight_txt_k=self.norm_added_k.weight)
            norms.append((self.norm_added_q, self.norm_added_k))
        q, k, v = buf.view(B, T + n, 3, self.heads, width // 3 // self.heads).unbind(2)
        cos, sin = image_rotary_emb
        turn = functools.partial(norm_rope_qk, q, k, weight_q=self.norm_q.weight, weight_k=self.norm_k.weight, cos=cos, sin=sin,
                                 **text)
        eps = {float(norm.eps) for pair in norms for norm in pair}
        if len(eps) == 1:
            turn(eps=eps.pop(), out=(q, k))
        else:  # a pass for each eps, of which every norm's rows are taken
            turned = {e: turn(eps=e) for e in eps}
            for rows, pair in zip((slice(T, None), slice(0, T)), norms):
                for i, (x, norm) in enumerate(zip((q, k), pair)):
                    x[:, rows] = turned[float(norm.eps)][i][:, rows]
        return q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)


def quantize_flux_model(model):
    """Rewrite ``model`` (a ``FluxTransformer`` on a CUDA device, not sharded) to 8-bit
    weights and activations, in place; returns it.  The 16-bit layers are given up when
    all 8-bit ones exist (half as much memory again until then), so a call that fails
    leaves the model as it was."""
    if not isinstance(model, FluxTransformer):
        raise TypeError("quantize_flux_model takes a flux_model.FluxTransformer; Int8Linear replaces single layers")
    if getattr(model, "int8", False):
        raise ValueError("the model is in 8 bits already")
    if getattr(model, "tp_world", None) is not None or model.sequence_parallel is not None:
        raise ValueError("a model sharded over GPUs cannot be quantised")
    if any(m.processor.__class__.__name__ == "PersistentFluxProcessor" for m in model.attention_modules()):
        raise ValueError("quantise the model outside persistent_flux_attention")
    if not model.x_embedder.weight.is_cuda:
        raise ValueError("quantize_flux_model needs the model on a CUDA device")
    if type(model.ops) is not NativeBlockOps:
        raise ValueError("the model's own block_ops would be replaced; 8-bit layers need those of this module")
    changes = []  # made when every layer exists: a failure on the way leaves the model as it was
    with torch.no_grad():
        for b in model.transformer_blocks:
            changes += [(b, "mod_img", Int8Linear(b.mod_img)), (b, "mod_txt", Int8Linear(b.mod_txt))]
            changes.append((b, "attn", Int8JointAttention(b.attn)))
            changes += [(ff, str(i), Int8Linear(ff[i])) for ff in (b.ff_img, b.ff_txt) for i in range(2)]
        for b in model.single_transformer_blocks:
            changes += [(b, "mod", Int8Linear(b.mod)), (b, "attn", Int8JointAttention(b.attn))]
            changes += [(b, "proj_mlp", Int8Linear(b.proj_mlp)), (b, "proj_out", Int8JoinedLinear(b.proj_out))]
    for owner, name, layer in changes:
        setattr(owner, name, layer)
    model.ops = Int8BlockOps()
    model.int8 = True
    return model.eval()


__all__ = ["quantize_flux_model", "Int8JointAttention", "Int8JoinedLinear", "Int8BlockOps"]
