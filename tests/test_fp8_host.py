"""The 8-bit block-scaled operators without a GPU: what the C entry points refuse (no kernel is launched), what they answer to empty
problems, the workspaces they ask for, and the layers' parameters."""

import ctypes

import pytest
import torch

from mlc_llm_amd import _lib, nn as layers, ops

P = ctypes.c_void_p
X, XS, W, WS, Y, Z = (P(0x1000 * i) for i in range(1, 7))


def _err():
    return _lib.lib().mi355gq_last_error().decode()


def _refused(code, text=None):
    assert code == _lib.ERR_ARG
    assert text is None or text in _err(), _err()


def _codes():
    ops_of = ops._MODEL_DTYPES
    return ops_of[torch.float16], ops_of[torch.float32], ops_of[torch.bfloat16]


def test_quantisers_check_their_arguments():
    f16, f32, bf16 = _codes()
    lib = _lib.lib()
    for name in ("mi355gq_fp8_quantize", "mi355gq_fp8_silu_mul_quantize"):
        fn = getattr(lib, name)
        _refused(fn(X, 4, 128, 9, Y, 128, WS, None), "model_dtype")
        _refused(fn(X, -1, 128, f16, Y, 128, WS, None), "shape")
        _refused(fn(X, 4, 1 << 40, f16, Y, 1 << 40, WS, None), "shape")
        _refused(fn(X, 4, 1 << 25, f16, Y, 1 << 25, WS, None), "shape")
        _refused(fn(X, 4, 130, f16, Y, 130, WS, None), "multiple of 16")
        _refused(fn(X, 4, 130, f16, Y, 128, WS, None), "multiple of 16")
        _refused(fn(None, 4, 128, f16, Y, 128, WS, None), "null")
        _refused(fn(P(0x1001), 4, 128, f16, Y, 128, WS, None), "aligned")
        _refused(fn(X, 4, 128, f32, P(0x5008), 128, WS, None), "aligned")
        assert fn(None, 0, 128, bf16, None, 128, None, None) == 0
    fn = lib.mi355gq_fp8_quantize_weight
    _refused(fn(W, 1, 128, 128, 7, Y, 128, WS, None), "model_dtype")
    _refused(fn(W, 1, -2, 128, f16, Y, 128, WS, None), "shape")
    _refused(fn(W, 1, 128, 129, f16, Y, 129, WS, None), "multiple of 16")
    _refused(fn(W, 2, 128, 128, f16, None, 128, WS, None), "null")
    assert fn(None, 0, 128, 128, f16, None, 128, None, None) == 0
    fn = lib.mi355gq_fp8_dequantize
    _refused(fn(W, 128, WS, 1, 128, 128, 0, 8, Y, None), "out_dtype")
    _refused(fn(W, 128, WS, 2, 128, 128, 1, f16, Y, None), "row_groups")
    _refused(fn(W, 112, WS, 1, 128, 128, 0, f16, Y, None), "multiple of 16")
    _refused(fn(W, 128, None, 1, 128, 128, 0, f16, Y, None), "null")
    assert fn(None, 128, None, 1, 0, 128, 0, f16, None, None) == 0


def test_products_check_their_arguments():
    f16, f32, bf16 = _codes()
    lib = _lib.lib()

    def linear(x=X, x_pitch=0, xs=None, w=W, w_pitch=128, ws=WS, bias=None, m=4, n=64, k=128, dtype=f16, out=f16, y=Y, space=Z, size=1 << 30):
        return lib.mi355gq_fp8_linear(x, x_pitch, xs, w, w_pitch, ws, bias, None, m, n, k, dtype, out, 0, y, space, size, None)

    _refused(linear(dtype=5), "model_dtype")
    _refused(linear(out=-1), "out_dtype")
    _refused(linear(k=0), "shape")
    _refused(linear(n=1 << 31), "shape")
    _refused(linear(w_pitch=120), "pitch")
    _refused(linear(k=130, w_pitch=128), "pitch")
    _refused(linear(xs=XS, x_pitch=64), "pitch")
    _refused(linear(w=None), "null")
    _refused(linear(y=None), "null")
    _refused(linear(w=P(0x3008)), "aligned")
    _refused(linear(bias=P(0x3001)), "aligned")
    _refused(linear(m=1 << 23), "rows")
    assert linear(x=None, w=None, ws=None, y=None, m=0) == 0
    assert linear(n=0, w=None) == 0
    assert linear(k=1 << 24, w_pitch=1 << 24) == _lib.ERR_UNSUPPORTED and "2^24" in _err()
    need = lib.mi355gq_fp8_linear_workspace_bytes(200, 64, 4096, 0)
    assert need >= 200 * 4096 + 4 * 200 * 32
    assert linear(m=200, k=4096, w_pitch=4096, size=need - 1) == _lib.ERR_WORKSPACE
    assert linear(m=200, k=4096, w_pitch=4096, space=None) == _lib.ERR_WORKSPACE
    _refused(linear(m=200, k=4096, w_pitch=4096, space=P(0x7008)), "aligned")
    assert lib.mi355gq_fp8_linear_workspace_bytes(0, 64, 128, 0) == 0 and lib.mi355gq_fp8_linear_workspace_bytes(-5, 64, 128, 0) == 0

    def grouped(x=X, xs=XS, x_rows=8, index=None, rows=8, w=W, indptr=Z, experts=2, n=64, k=128, pitch=128, out=f16):
        return lib.mi355gq_fp8_group_gemm(x, pitch, xs, x_rows, index, rows, w, pitch, WS, indptr, experts, n, k, out, 0, Y, None)

    _refused(grouped(out=4), "out_dtype")
    _refused(grouped(experts=0), "shape")
    _refused(grouped(experts=513), "shape")
    _refused(grouped(pitch=72), "pitch")
    _refused(grouped(x_rows=7), "without an index")
    _refused(grouped(indptr=None), "null")
    _refused(grouped(xs=P(0x2002)), "aligned")
    _refused(grouped(rows=1 << 30, x_rows=1 << 30), "rows")
    assert grouped(rows=0, x=None) == 0
    assert grouped(index=Y, x_rows=1 << 26) == _lib.ERR_UNSUPPORTED and "4 GiB" in _err()
    assert grouped(k=1 << 24, pitch=1 << 24) == _lib.ERR_UNSUPPORTED


def test_routing_and_the_layer_check_their_arguments():
    f16, f32, bf16 = _codes()
    lib = _lib.lib()

    def gating(logits=X, t=4, e=8, k=2, scoring=_lib.SCORE_SOFTMAX, groups=1, top=1, dtype=f16, ids=Y, weights=Z):
        return lib.mi355gq_moe_gating(logits, None, t, e, k, scoring, groups, top, 1, 1.0, dtype, weights, ids, None)

    for bad in ({"dtype": 3}, {"scoring": 2}, {"t": -1}, {"e": 0}, {"e": 513}, {"k": 0}, {"k": 9}, {"e": 64, "k": 33}, {"groups": 3},
                {"groups": 65, "e": 130}, {"groups": 4, "top": 5}, {"groups": 4, "top": 0}, {"groups": 4, "top": 1, "k": 3},
                {"logits": None}, {"ids": None}, {"weights": P(0x6002)}, {"logits": P(0x1001)}):
        _refused(gating(**bad))
    assert gating(t=0, logits=None, ids=None, weights=None) == 0
    plan = lib.mi355gq_moe_plan
    _refused(plan(X, 4, 0, 8, Y, Z, W, None))
    _refused(plan(X, 4, 2, 513, Y, Z, W, None))
    _refused(plan(X, 1 << 30, 4, 8, Y, Z, W, None))
    _refused(plan(None, 4, 2, 8, Y, Z, W, None), "null")
    _refused(plan(X, 4, 2, 8, Y, Z, None, None), "null")
    _refused(plan(P(0x1002), 4, 2, 8, Y, Z, W, None), "aligned")

    def layer(x=X, t=4, hidden=256, inter=128, experts=8, k=2, p13=256, p2=128, dtype=f16, space=Z, size=1 << 30, ids=Y):
        return lib.mi355gq_fp8_moe(x, t, hidden, inter, experts, k, XS, ids, W, p13, WS, W, p2, WS, dtype, Y, space, size, None)

    for bad in ({"dtype": f32}, {"hidden": 200, "p13": 208}, {"inter": 100, "p2": 112}, {"experts": 0}, {"experts": 513}, {"k": 33}, {"t": -1},
                {"p13": 128}, {"p2": 100}, {"t": 1 << 25}, {"x": None}, {"ids": None}, {"x": P(0x1008)}, {"space": P(0x7004)}):
        _refused(layer(**bad))
    assert layer(t=0, x=None) == 0
    need = lib.mi355gq_fp8_moe_workspace_bytes(4, 256, 128, 8, 2)
    assert need > 0 and layer(size=need - 1) == _lib.ERR_WORKSPACE and layer(space=None) == _lib.ERR_WORKSPACE
    assert lib.mi355gq_fp8_moe_workspace_bytes(4, 250, 128, 8, 2) == 0


def test_operators_refuse_cpu_tensors():
    x, w = torch.zeros(2, 128, dtype=torch.float16), torch.zeros(64, 128, dtype=torch.float8_e4m3fn)
    scale = torch.zeros(1, 1)
    calls = [lambda: ops.fp8_quantize(x), lambda: ops.fp8_silu_mul_quantize(x), lambda: ops.fp8_quantize_weight(x),
             lambda: ops.fp8_dequantize(w, scale), lambda: ops.fp8_linear(x, w, scale), lambda: ops.fp8_linear((w, scale), w, scale),
             lambda: ops.fp8_group_gemm(w, scale, None, w[None], scale[None], torch.zeros(2, dtype=torch.int32)),
             lambda: ops.moe_gating(x, 2), lambda: ops.moe_plan(torch.zeros(2, 2, dtype=torch.int32), 4),
             lambda: ops.fp8_moe(x, x, w[None], scale[None], w[None], scale[None], 1)]
    for call in calls:
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_layers_hold_weights_of_padded_rows():
    linear = layers.Fp8Linear(200, 300, bias=True, dtype=torch.bfloat16)
    assert linear.q_weight.shape == (300, 200) and linear.q_weight.stride() == (208, 1) and linear.q_weight.dtype == torch.float8_e4m3fn
    assert linear.q_scale.shape == (3, 2) and linear.q_scale.dtype == torch.float32 and linear.bias.dtype == torch.bfloat16
    assert layers.Fp8Linear(128, 64, bias=False).bias is None
    moe = layers.Fp8MoE(256, 272, 5, 2, scoring="sigmoid", score_bias=True)
    assert moe.e1_e3.q_weight.shape == (5, 544, 256) and moe.e1_e3.q_scale.shape == (5, 5, 2)
    assert moe.e2.q_weight.shape == (5, 256, 272) and moe.e2.q_scale.shape == (5, 2, 3) and moe.score_bias.shape == (5,)
    assert sorted(moe.state_dict()) == ["e1_e3.q_scale", "e1_e3.q_weight", "e2.q_scale", "e2.q_weight", "score_bias"]
    assert not any(p.requires_grad for p in moe.parameters())
    with pytest.raises(ValueError, match="expected"):
        moe.load_experts(torch.zeros(5, 544, 128), torch.zeros(5, 256, 272))


def test_layer_workspace_holds_what_the_call_uses():
    lib = _lib.lib()
    size = lib.mi355gq_fp8_moe_workspace_bytes

    def pieces(t, hidden, inter, experts, k):
        """x and the activation in e4m3 with their scales, the plan, the second product in float32; nine pieces of multiples of 256."""
        slots = t * k
        return (t * hidden + slots * inter + 4 * (t * -(-hidden // 128) + slots * -(-inter // 128) + 2 * slots + experts + 1 + slots * hidden) + 9 * 256)

    # gate and up in float32, the largest piece by far, where the activation is not quantised as it comes up: 8 slots * inter bytes
    for case in ((2048, 4096, 14336, 8, 2), (2048, 2048, 768, 128, 8), (16, 2048, 768, 128, 8), (2, 256, 128, 4, 1)):
        assert 0 < size(*case) <= pieces(*case)
    for case in ((2048, 4096, 14320, 8, 2), (16, 2048, 144, 64, 6), (1, 2048, 1408, 64, 6), (2, 16384, 131072, 1, 1)):
        assert pieces(*case) - 9 * 256 <= size(*case) - 8 * case[0] * case[4] * case[2] <= pieces(*case)
    # rows of gate and up so far apart that an expert's reach 4 GiB
    f16 = _codes()[0]
    need = size(40, 256, 256, 2, 1)
    pitch = (1 << 23) + 16
    for given in (need, need + 8 * 40 * 256 - 1):
        assert lib.mi355gq_fp8_moe(X, 40, 256, 256, 2, 1, XS, Y, W, pitch, WS, W, 256, WS, f16, Y, Z, given, None) == _lib.ERR_WORKSPACE


class _OnGpu(torch.Tensor):
    """A CPU tensor that passes for one on the GPU, for checks that look at strides alone."""

    is_cuda = True


def _strided(nbytes, shape, strides, offset=0):
    return torch.zeros(nbytes, dtype=torch.uint8).view(torch.float8_e4m3fn).as_strided(shape, strides, offset).as_subclass(_OnGpu)


@pytest.mark.parametrize("nbytes,shape,strides,offset,pitch", [
    (5 * 208, (5, 200), (208, 1), 0, 208), (4 * 208 + 200, (5, 200), (208, 1), 0, None), (4 * 208 + 207, (5, 200), (208, 1), 0, None),
    (5 * 208 + 16, (5, 200), (208, 1), 16, 208), (5 * 208 + 15, (5, 200), (208, 1), 16, None), (4 * 208 + 192, (5, 192), (208, 1), 0, 208),
    (200, (1, 200), (208, 1), 0, None), (208, (1, 200), (208, 1), 0, 208), (208, (1, 200), (200, 1), 0, 208),
    # the last row of a wider matrix, some of its columns: what lies behind them in the pitch is not theirs and is not needed
    (4 * 4096, (1, 88), (4096, 1), 3 * 4096 + 4000, 96), (4 * 130, (1, 128), (130, 1), 0, 128),
    (3 * 208, (3, 1, 200), (208, 208, 1), 0, 208), (2 * 208 + 200, (3, 1, 200), (208, 208, 1), 0, None), (3 * 512, (3, 1, 128), (512, 7, 1), 0, 512),
    (6 * 112, (3, 2, 100), (224, 112, 1), 0, 112), (6 * 112 - 1, (3, 2, 100), (224, 112, 1), 0, None), (3 * 240, (3, 2, 100), (240, 112, 1), 0, None),
    (5 * 200, (5, 200), (200, 1), 0, None), (5 * 208, (5, 200), (208, 0), 0, None), (208, (5, 200), (0, 1), 0, None), (0, (0, 200), (200, 1), 0, 208)])
def test_rows_of_e4m3_lie_in_their_storage(nbytes, shape, strides, offset, pitch):
    if pitch is None:
        with pytest.raises(ValueError, match="of storage|multiple of 16 bytes apart"):
            ops._chk_fp8(_strided(nbytes, shape, strides, offset), "q", len(shape))
    else:
        assert ops._chk_fp8(_strided(nbytes, shape, strides, offset), "q", len(shape)) == pitch


@pytest.mark.parametrize("t,k", [((1 << 31) - 300, 1), ((1 << 31) - 1500, 1), ((1 << 30) - 600, 2)])
def test_plan_refuses_slots_that_its_waves_cannot_count(t, k):
    # a wave's run is a multiple of 64 slots, and the last ones end behind the slots: past 2^31 there a wave would see none of its own
    _refused(_lib.lib().mi355gq_moe_plan(X, t, k, 8, Y, Z, W, None), "moe_plan")


def test_plan_counts_in_32_bits():
    largest = (1 << 31) - 256 - 2048
    for slots in (largest, largest - 1, largest // 2):
        waves = 16
        per_wave = ((slots + waves - 1) // waves + 63) // 64 * 64
        begin, end = (waves - 1) * per_wave, min(waves * per_wave, slots)
        assert waves * per_wave < 2**31 and begin + 4 * 64 < 2**31 and end + 64 + 63 < 2**31
