"""``Int8Linear`` and the 8-bit FLUX model after casts, moves and reloads: the outputs
are those of the same codes."""

from __future__ import annotations

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _linear(k, n, bias=True):
    torch.manual_seed(k + n)
    return torch.nn.Linear(k, n, bias=bias, device="cuda", dtype=BF16)


@pytest.mark.parametrize("k,n", [(64, 40), (1001, 130), (1000, 1)])
@pytest.mark.parametrize("bias", [True, False])
def test_layer_after_casts_moves_and_reloads(k, n, bias):
    import hilberta_b200 as hb

    linear = _linear(k, n, bias)
    weight = hb.quantize_rows(linear.weight.detach())
    x = torch.randn(33, k, device="cuda").to(BF16)
    with torch.inference_mode():
        want = hb.int8_linear(x, weight, linear.bias)
        want16 = hb.int8_linear(x.to(FP16), weight, None if linear.bias is None else linear.bias.to(FP16))
        layer = hb.Int8Linear(linear)
        assert torch.equal(layer(x), want)
        assert torch.equal(layer.to(BF16)(x), want) and torch.equal(layer.float()(x), want)
        assert torch.equal(copy.deepcopy(layer).half()(x.to(FP16)), want16)
        assert torch.equal(copy.deepcopy(layer)(x), want)
        assert torch.equal(layer.cpu().cuda()(x), want) and torch.equal(layer.to("cpu", FP16).to("cuda")(x.to(FP16)), want16)
        for assign in (False, True):
            state = {name: t.contiguous() for name, t in hb.Int8Linear(linear).state_dict().items()}
            other = hb.Int8Linear(_linear(k, n, bias).requires_grad_(False))
            other.values.zero_()
            other.load_state_dict(state, assign=assign)
            assert torch.equal(other(x), want)
        with pytest.raises(ValueError, match="CUDA"):
            hb.Int8Linear(linear).cpu()(x)


def test_quantised_model_in_the_other_type():
    """The whole model cast and moved: every 8-bit layer keeps its codes and answers in the new type."""
    from hilberta_b200.flux_int8 import quantize_flux_model
    from hilberta_b200.flux_model import FluxTransformer, step_inputs
    from hilberta_b200.int8 import Int8Linear

    torch.manual_seed(0)
    model = quantize_flux_model(
        FluxTransformer(num_double=1, num_single=1, dim=256, heads=2, text_dim=64, pooled_dim=32, device="cuda"))
    codes = {name: (m.values.clone(), m.scales.clone()) for name, m in model.named_modules() if isinstance(m, Int8Linear)}
    inputs = lambda dtype: step_inputs(8, 16, "cuda", seed=3, text_dim=64, pooled_dim=32, dtype=dtype)  # noqa: E731
    with torch.inference_mode():
        want = model(**inputs(BF16)).sample
        half = model.half()(**inputs(FP16)).sample
        assert half.dtype == FP16 and half.isfinite().all()
        assert torch.equal(model.cpu().cuda()(**inputs(FP16)).sample, half)
        model.bfloat16()
        for name, m in model.named_modules():
            if isinstance(m, Int8Linear):
                assert torch.equal(m.values, codes[name][0]) and torch.equal(m.scales, codes[name][1]) and m.dtype == BF16
        assert model(**inputs(BF16)).sample.isfinite().all() and want.shape == half.shape
