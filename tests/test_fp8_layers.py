"""The layers on 8-bit block-scaled weights when a model is copied, moved, saved and cast, without a GPU."""

import copy
import io

import pytest
import torch

from mlc_llm_amd import nn as layers


def _filled(t):
    t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(t.numel())))


def _same(a, b):
    return torch.equal(a.float(), b.float())


def _linear(n=40, k=200):
    layer = layers.Fp8Linear(k, n, bias=True)
    for p in layer.parameters():
        _filled(p.data)
    return layer


def _saved(layer):
    file = io.BytesIO()
    torch.save(layer, file)
    file.seek(0)
    return torch.load(file, weights_only=False)  # (written above)


def _assigned(layer):
    other = layers.Fp8Linear(layer.in_features, layer.out_features)
    other.load_state_dict({name: v.clone() for name, v in layer.state_dict().items()}, assign=True)
    return other


def _loaded(layer):
    other = layers.Fp8Linear(layer.in_features, layer.out_features)
    other.load_state_dict(layer.state_dict())
    return other


WAYS = {"deepcopy": copy.deepcopy, "apply": lambda layer: copy.deepcopy(layer)._apply(torch.clone), "save": _saved, "assign": _assigned,
        "load": _loaded, "inside": lambda layer: copy.deepcopy(torch.nn.Sequential(torch.nn.ModuleList([layer])))[0][0],
        "to": lambda layer: copy.deepcopy(layer).to("cpu")}


@pytest.mark.parametrize("way", sorted(WAYS))
@pytest.mark.parametrize("n,k", [(40, 200), (1, 10), (3, 112), (130, 257)])
def test_rows_stay_a_multiple_of_16_bytes_apart(way, n, k):
    layer = _linear(n, k)
    other = WAYS[way](layer)
    pitch = -(-k // 16) * 16
    assert other is not layer and other.q_weight.shape == (n, k) and other.q_weight.stride() == (pitch, 1)
    assert other.q_weight.untyped_storage().nbytes() >= n * pitch and not other.q_weight.requires_grad
    assert isinstance(other.q_weight, torch.nn.Parameter) and sorted(other.state_dict()) == ["bias", "q_scale", "q_weight"]
    for name, v in layer.state_dict().items():
        assert _same(other.state_dict()[name], v) and other.state_dict()[name].dtype == v.dtype


def test_rows_of_a_layer_on_another_device():
    linear = _linear().to("meta")
    assert linear.q_weight.is_meta and linear.q_weight.stride() == (208, 1)
    assert linear.to_empty(device="cpu").q_weight.stride() == (208, 1)
    moe = copy.deepcopy(layers.Fp8MoE(250, 144, 3, 2))
    assert moe.e1_e3.q_weight.stride() == (288 * 256, 256, 1) and moe.e2.q_weight.stride() == (250 * 144, 144, 1)
    assert moe.to("meta").e1_e3.q_weight.stride() == (288 * 256, 256, 1)


CASTS = {"half": lambda m: m.half(), "bfloat16": lambda m: m.to(torch.bfloat16), "float": lambda m: m.float(), "double": lambda m: m.double(),
         "device and type": lambda m: m.to("cpu", torch.bfloat16), "type": lambda m: m.type(torch.float16), "meta": lambda m: m.to("meta", torch.float16),
         "inside": lambda m: torch.nn.Sequential(torch.nn.Linear(3, 3), m).half()[1]}


@pytest.mark.parametrize("cast", sorted(CASTS))
def test_a_cast_leaves_weights_scales_and_the_choice_bias(cast):
    linear, moe = _linear(), layers.Fp8MoE(256, 144, 3, 2, scoring="sigmoid", score_bias=True)
    for p in moe.parameters():
        _filled(p.data)
    before = [{name: v.clone() for name, v in m.state_dict().items()} for m in (linear, moe)]
    other = CASTS[cast](linear), CASTS[cast](moe)
    assert other[0].q_weight.stride() == (208, 1)
    bias_type = {"bfloat16": torch.bfloat16, "device and type": torch.bfloat16, "float": torch.float32, "double": torch.float64}.get(cast, torch.float16)
    assert other[0].bias.dtype == bias_type  # this one has the model's type
    for m, was in zip(other, before):
        for name, v in m.state_dict().items():
            if name != "bias":
                assert v.dtype == was[name].dtype and (v.is_meta or _same(v, was[name]))
