"""The FLUX.1-architecture model in 8 bits (hilberta_b200/flux_int8.py).

Against the 16-bit model: a row of normal values has its largest near 4 of their
deviation, so a code's rounding error is 4 / 127 / sqrt(12) = 0.9 % of it; weights and
activations together 1.3 % of a product.  Five layers of at most four products in a
row, added as independent errors: sqrt(20) * 1.3 % = 5.8 % of the prediction.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _models():
    import copy

    from hilberta_b200.flux_int8 import quantize_flux_model
    from hilberta_b200.flux_model import FluxTransformer

    torch.manual_seed(0)
    model = FluxTransformer(num_double=2, num_single=3, dim=256, heads=2, text_dim=64, pooled_dim=32, device="cuda")
    with torch.no_grad():
        for m in model.modules():
            if isinstance(m, torch.nn.Linear):
                m.bias.normal_(0.0, 0.1)
    quantised = copy.deepcopy(model)
    assert quantize_flux_model(quantised) is quantised
    return model, quantised


def _inputs(plan, batch=2):
    from hilberta_b200.flux_model import step_inputs

    x = step_inputs(plan.grid_size, plan.text_tokens, "cuda", batch=batch, seed=3, text_dim=64, pooled_dim=32)
    x["timestep"] = torch.tensor([0.3, 0.9][:batch], device="cuda")
    return x


def _rel(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def _run(model, plan, x, **kw):
    from hilberta_b200 import persistent_flux_attention

    with torch.inference_mode(), persistent_flux_attention(model, plan, **kw) as info:
        out = model(**x).sample
    return out, info


def test_backends_dense_and_16_bit_model():
    import hilberta_b200 as hb

    plan = hb.bridge_k_plan(4, 1, False, grid_size=32)
    model, quantised = _models()
    x = _inputs(plan)
    paired, info = _run(quantised, plan, x, backend="paired")
    assert torch.isfinite(paired).all() and info["layer_calls"] == [1] * 5
    # the same quantised layers around the attention: only the attention's own rounding
    # differs, and the quantisation steps it flips
    assert _rel(_run(quantised, plan, x, backend="sdpa_reference")[0], paired) < 2e-2
    assert torch.equal(_run(quantised, plan, x, backend="sparse")[0], paired)
    assert _rel(paired, _run(model, plan, x, backend="paired")[0]) < 5.8e-2
    with torch.inference_mode():
        dense, dense16 = quantised(**x).sample, model(**x).sample
    assert _rel(dense, dense16) < 5.8e-2
    assert hb.device_status() == 0


def test_batch_entry_alone():
    import hilberta_b200 as hb

    plan = hb.bridge_k_plan(4, 1, False, grid_size=32)
    _, quantised = _models()
    x = _inputs(plan)
    both, _ = _run(quantised, plan, x, backend="paired")
    one = {k: v[1:] if k in ("hidden_states", "encoder_hidden_states", "pooled_projections", "timestep", "guidance") else v
           for k, v in x.items()}
    # the 16-bit embedders and the attention may round otherwise at another batch size
    assert _rel(_run(quantised, plan, one, backend="paired")[0], both[1:]) < 2e-2


def test_captured_blocks():
    """Double- and single-stream blocks captured into a graph and replayed on new
    inputs equal the eager blocks."""
    from hilberta_b200.flux_model import image_ids, rotary_3axis

    _, quantised = _models()
    g = torch.Generator(device="cuda").manual_seed(1)
    img, txt, temb = (torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16) for s in ((1, 64, 256), (1, 24, 256), (1, 256)))
    rot = rotary_3axis(torch.cat([torch.zeros(24, 3, dtype=torch.int64, device="cuda"), image_ids(8, "cuda")]), (16, 56, 56))

    def blocks(img, txt):
        for b in quantised.transformer_blocks:
            img, txt = b(img, txt, temb, rot, quantised.ops)
        x = torch.cat([txt, img], dim=1)
        for b in quantised.single_transformer_blocks:
            x = b(x, temb, rot, quantised.ops)
        return x

    with torch.inference_mode():
        static = img.clone(), txt.clone()
        blocks(*(t.clone() for t in static))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = blocks(*(t.clone() for t in static))
        for t in static:
            t.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, blocks(*(t.clone() for t in static)))


def test_layers_share_the_joined_weights():
    from hilberta_b200.int8 import Int8Linear

    model, quantised = _models()
    a, b = model.transformer_blocks[0].attn, quantised.transformer_blocks[0].attn
    x = torch.randn(2, 9, 256, device="cuda").to(torch.bfloat16)
    with torch.inference_mode():
        for name in ("to_q", "to_k", "to_v", "add_q_proj", "add_k_proj", "add_v_proj"):
            assert torch.equal(getattr(b, name)(x), Int8Linear(getattr(a, name))(x))
        joined = b.to_qkv(x)
        assert torch.equal(joined[..., 256:512], b.to_k(x))
    assert b.to_k.values.data_ptr() == b.to_qkv.values[256:].data_ptr()


def test_refusals():
    from hilberta_b200.flux_int8 import quantize_flux_model

    _, quantised = _models()
    with pytest.raises(ValueError, match="already"):
        quantize_flux_model(quantised)
    attn = quantised.transformer_blocks[0].attn
    h = torch.zeros(1, 64, 256, dtype=torch.bfloat16, device="cuda")
    with torch.inference_mode(), pytest.raises(ValueError, match="rotary"):
        attn.joint_qkv(h, None, None)
