"""The layers on 16-bit weights: their parameters on the CPU, and on the GPU the operators' own results."""

import copy

import pytest
import torch

from mlc_llm_amd import nn as layers, ops


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_parameters(dtype):
    src = torch.nn.Linear(24, 10, dtype=dtype)
    layer = layers.DenseLinear.from_linear(src, "gelu")
    assert layer.weight.data_ptr() == src.weight.data_ptr() and layer.bias.data_ptr() == src.bias.data_ptr()
    assert (layer.in_features, layer.out_features, layer.activation) == (24, 10, "gelu") and not layer.weight.requires_grad
    gated = layers.DenseGatedLinear.from_linear(src)
    assert (gated.out_features, gated.activation) == (5, "silu") and gated.weight.shape == (10, 24)
    with pytest.raises(ValueError, match="gate and up"):
        layers.DenseGatedLinear.from_linear(torch.nn.Linear(8, 3))
    assert layers.DenseLinear.from_linear(torch.nn.Linear(8, 4, bias=False)).bias is None
    fresh = layers.DenseGatedLinear(16, 8, dtype=dtype)
    assert fresh.weight.shape == (16, 16) and fresh.bias.shape == (16,) and fresh.weight.dtype == dtype
    moe = layers.DenseMoE(32, 16, 4, 2, score_bias=True, dtype=dtype)
    assert sorted(moe.state_dict()) == ["e1_e3.weight", "e2.weight", "score_bias"]
    assert moe.e1_e3.weight.shape == (4, 32, 32) and moe.e2.weight.shape == (4, 32, 16) and moe.e2.weight.dtype == dtype
    moe.score_bias.data[1] = 0.3333333
    other = torch.bfloat16 if dtype == torch.float16 else torch.float16
    for cast in (lambda m: m.to(other), lambda m: m.half(), copy.deepcopy):
        got = cast(copy.deepcopy(moe))
        assert got.score_bias.dtype == torch.float32 and got.score_bias[1] == moe.score_bias[1]
    assert moe.to(other).e1_e3.weight.dtype == other


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_layers_are_the_operators(dtype):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 5, 64, generator=g).to(dtype).cuda()
    src = torch.nn.Linear(64, 48, dtype=dtype, device="cuda")
    layer = layers.DenseLinear.from_linear(src, "relu", torch.float32)
    r = torch.randn(2, 5, 48, generator=g).to(dtype).cuda()
    assert torch.equal(layer(x, r), ops.dense_linear(x, src.weight.detach(), src.bias.detach(), "relu", r, torch.float32))
    assert torch.equal(layers.DenseGatedLinear.from_linear(src)(x), ops.dense_linear_gated(x, src.weight.detach(), src.bias.detach()))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [0, 1, 64, 65, 150])
def test_expert_layer_of_any_number_of_tokens(tokens):
    g = torch.Generator().manual_seed(tokens)
    moe = layers.DenseMoE(64, 40, 16, 3, scoring="sigmoid", score_bias=True, num_groups=4, top_groups=2, routed_scale=2.0, dtype=torch.bfloat16,
                          device="cuda")
    for p in (moe.e1_e3.weight, moe.e2.weight):
        p.data.copy_(torch.randn(p.shape, generator=g) / 8)
    moe.score_bias.data.copy_(torch.randn(16, generator=g) / 10)
    x, gate = torch.randn(1, tokens, 64, generator=g).bfloat16().cuda(), torch.randn(tokens, 16, generator=g).cuda()
    y = moe(x, gate)
    assert y.shape == x.shape
    for i in range(0, tokens, 64):
        part = ops.dense_moe(x[0, i : i + 64], gate[i : i + 64], moe.e1_e3.weight, moe.e2.weight, 3, scoring="sigmoid", bias=moe.score_bias,
                             num_groups=4, top_groups=2, scale=2.0)
        assert torch.equal(y[0, i : i + 64], part)


@pytest.mark.parametrize("shape", [(70, 4), (128, 4), (63, 4), (0, 4), (64,), (1, 64, 4), (64, 5)])
@pytest.mark.parametrize("tokens", [0, 64, 128])
def test_expert_layer_wants_a_row_of_logits_a_token(tokens, shape):
    """Rows of logits that no token goes with are refused, whatever runs the layer cuts its tokens into."""
    moe = layers.DenseMoE(8, 8, 4, 2)
    if shape == (tokens, 4):
        return
    with pytest.raises(ValueError, match=rf"gate \({', '.join(map(str, shape))},?\) for {tokens} tokens of 4 experts"):
        moe(torch.zeros(tokens, 8, dtype=torch.float16), torch.zeros(shape))
