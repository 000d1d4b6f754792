"""The operators on 16-bit weights without a GPU: what the C entry points and the Python ones refuse (no kernel is launched), and what
they answer to empty problems."""

import ctypes

import pytest
import torch

from mlc_llm_amd import _lib, ops

P = ctypes.c_void_p
X, W, B, R, Y, S = (P(0x10000 * i) for i in range(1, 7))
F16, F32, BF16 = _lib.F16, _lib.F32, _lib.BF16


def _refused(code, text, expect=_lib.ERR_ARG):
    assert code == expect
    assert text in _lib.lib().mi355gq_last_error().decode(), _lib.lib().mi355gq_last_error()


def test_products_check_their_arguments():
    def linear(x=X, w=W, b=B, r=R, m=4, n=64, k=128, act=0, dt=F16, out=F16, y=Y):
        return _lib.lib().mi355gq_dense_linear(x, w, b, r, m, n, k, act, dt, out, y, None, 0, None)

    def gated(x=X, w=W, b=B, m=4, n=64, k=128, act=2, dt=F16, out=F16, y=Y):
        return _lib.lib().mi355gq_dense_linear_gated(x, w, b, m, n, k, act, dt, out, y, None, 0, None)

    for fn in (linear, gated):
        _refused(fn(dt=F32, out=F32), "model_dtype")
        _refused(fn(dt=7), "model_dtype")
        _refused(fn(dt=F16, out=BF16), "out_dtype")
        _refused(fn(dt=BF16, out=F16), "out_dtype")
        _refused(fn(act=5), "activation")
        _refused(fn(act=-1), "activation")
        _refused(fn(m=-1), "shape")
        _refused(fn(n=-1), "shape")
        _refused(fn(k=0), "shape")
        _refused(fn(m=1 << 31), "shape")
        _refused(fn(n=1 << 31), "shape")
        _refused(fn(k=1 << 31), "shape")
        _refused(fn(k=1 << 23), "K=8388608", _lib.ERR_UNSUPPORTED)
        _refused(fn(x=None), "null")
        _refused(fn(w=None), "null")
        _refused(fn(y=None), "null")
        _refused(fn(x=P(0x10001)), "aligned")
        _refused(fn(b=P(0x10001)), "aligned")
        _refused(fn(out=F32, y=P(0x10002)), "aligned")
        assert fn(m=0, x=None, y=None) == 0
        assert fn(n=0, w=None, y=None) == 0
    _refused(linear(r=P(0x10001)), "aligned")
    _refused(gated(n=(1 << 30)), "shape")  # 2^31 rows of W
    size = _lib.lib().mi355gq_dense_linear_workspace_bytes
    assert size(0, 64, 64, 0) == size(64, 0, 64, 1) == size(64, 64, 0, 0) == size(-1, 64, 64, 0) == size(1 << 40, 64, 64, 0) == 0
    assert all(size(m, n, k, g) >= 0 for m in (1, 40, 5000) for n in (1, 4096) for k in (8, 4096) for g in (0, 1))


def test_expert_layer_checks_its_arguments():
    need = _lib.lib().mi355gq_dense_moe_workspace_bytes(4, 64, 32, 8, 2)
    assert need >= 2 * 4 * 2 * 32 * 2

    def moe(x=X, lg=B, sb=None, t=4, h=64, i=32, e=8, k=2, sc=0, g=1, tg=1, ldt=F32, w13=W, w2=R, act=2, dt=F16, out=Y, ws=S, size=need):
        return _lib.lib().mi355gq_dense_moe(x, lg, sb, t, h, i, e, k, sc, g, tg, 1, 1.0, ldt, w13, w2, act, dt, out, ws, size, None)

    _refused(moe(dt=F32), "model_dtype")
    _refused(moe(ldt=5), "logits_dtype")
    _refused(moe(act=9), "activation")
    _refused(moe(sc=2), "scoring")
    for bad in ({"t": -1}, {"h": 60}, {"h": 0}, {"i": 12}, {"e": 0}, {"e": 513}, {"k": 0}, {"k": 9}, {"k": 33, "e": 64}, {"h": 1 << 23}, {"i": 1 << 23}):
        _refused(moe(**bad), "multiples of 8")
    _refused(moe(g=3), "groups")
    _refused(moe(g=4, tg=5), "groups")
    _refused(moe(g=8, tg=1), "cannot give 2")
    _refused(moe(t=65), "64 tokens at most", _lib.ERR_UNSUPPORTED)
    _refused(moe(t=64, i=(1 << 23) - 256, e=64, k=32), "3 GiB", _lib.ERR_UNSUPPORTED)
    for name in ("x", "lg", "w13", "w2", "out"):
        _refused(moe(**{name: None}), "null")
    for name in ("x", "w13", "w2", "out"):
        _refused(moe(**{name: P(0x10008)}), "misaligned")
    _refused(moe(lg=P(0x10002)), "misaligned")
    _refused(moe(sb=P(0x10002)), "misaligned")
    _refused(moe(ws=P(0x10008)), "workspace")
    _refused(moe(size=need - 1), "needed", _lib.ERR_WORKSPACE)
    _refused(moe(ws=None), "needed", _lib.ERR_WORKSPACE)
    assert moe(t=0, x=None, ws=None) == 0
    size = _lib.lib().mi355gq_dense_moe_workspace_bytes
    assert size(0, 64, 32, 8, 2) == size(65, 64, 32, 8, 2) == size(4, 60, 32, 8, 2) == 0


def test_python_refusals():
    x, w = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(32, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="must live on the GPU"):
        ops.dense_linear(x, w)
    with pytest.raises(TypeError, match="expected a torch.Tensor"):
        ops.dense_linear([1.0], w)
    with pytest.raises(ValueError, match="must live on the GPU"):
        ops.dense_linear_gated(x, w)


@pytest.mark.gpu
def test_python_refusals_of_tensors():
    def t(*shape, dtype=torch.float16):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    x, w = t(4, 64), t(32, 64)
    for fn in (ops.dense_linear, ops.dense_linear_gated):
        with pytest.raises(TypeError, match="x: dtype"):
            fn(x.float(), w.float())
        with pytest.raises(TypeError, match="weight: dtype"):
            fn(x, w.bfloat16())
        with pytest.raises(ValueError, match="for a weight of"):
            fn(x, t(32, 72))
        with pytest.raises(ValueError, match="for a weight of"):
            fn(t(4, 0), t(32, 0))
        with pytest.raises(ValueError, match=r"\[N, K\]"):
            fn(x, t(2, 32, 64))
        with pytest.raises(ValueError, match="x: must be contiguous"):
            fn(t(64, 4).t(), w)
        with pytest.raises(ValueError, match="weight: must be contiguous"):
            fn(x, t(64, 32).t())
        with pytest.raises(ValueError, match="bias shape"):
            fn(x, w, bias=t(31))
        with pytest.raises(TypeError, match="bias: dtype"):
            fn(x, w, bias=t(32, dtype=torch.float32))
        with pytest.raises(ValueError, match="activation 'tanh'"):
            fn(x, w, activation="tanh")
        with pytest.raises(ValueError, match="activation 3"):
            fn(x, w, activation=3)
        with pytest.raises(TypeError, match="out_dtype"):
            fn(x, w, out_dtype=torch.bfloat16)
        with pytest.raises(ValueError, match="must live on the GPU"):
            fn(x, w, bias=torch.zeros(32, dtype=torch.float16))
    with pytest.raises(ValueError, match="split into gate and up"):
        ops.dense_linear_gated(x, t(33, 64))
    with pytest.raises(ValueError, match="residual shape"):
        ops.dense_linear(x, w, residual=t(4, 31))
    with pytest.raises(TypeError, match="residual: dtype"):
        ops.dense_linear(x, w, residual=t(4, 32, dtype=torch.float32))
    with pytest.raises(ValueError, match="out shape"):
        ops.dense_linear(x, w, out=t(32, 4))
    with pytest.raises(TypeError, match="out: dtype"):
        ops.dense_linear(x, w, out=t(4, 32), out_dtype=torch.float32)
    square = t(64, 64)
    for out in (x[:4], square[4:8], square[:4]):
        with pytest.raises(ValueError, match="out: shares memory"):
            ops.dense_linear(x, square, out=out)
    pair = t(8, 32)
    w13, w2, logits = t(8, 64, 64), t(8, 64, 32), t(4, 8, dtype=torch.float32)
    ops.dense_moe(x, logits, w13, w2, 2)
    for bad, err, text in (((x.float(), logits, w13, w2), TypeError, "x: dtype"), ((x, logits.double(), w13, w2), TypeError, "logits: dtype"),
                           ((x, logits, w13.bfloat16(), w2), TypeError, "w13: dtype"), ((x, logits, w13[0], w2), ValueError, "dimensions"),
                           ((x, logits, w13[:7], w2), ValueError, "do not belong together"), ((x, logits[:3], w13, w2), ValueError, "logits shape"),
                           ((t(4, 72), logits, w13, w2), ValueError, "do not belong together")):
        with pytest.raises(err, match=text):
            ops.dense_moe(*bad, 2)
    with pytest.raises(ValueError, match="bias shape"):
        ops.dense_moe(x, logits, w13, w2, 2, bias=t(7, dtype=torch.float32))
    with pytest.raises(ValueError, match="scoring"):
        ops.dense_moe(x, logits, w13, w2, 2, scoring="relu")
    with pytest.raises(ValueError, match="activation"):
        ops.dense_moe(x, logits, w13, w2, 2, activation="swish")
    with pytest.raises(ValueError, match="out: shares memory"):
        ops.dense_linear(x, w, residual=pair[:4], out=pair[1:5])
