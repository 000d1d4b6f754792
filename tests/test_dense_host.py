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
    with pytest.raises(ValueError, match="out: shares memory"):
        ops.dense_linear(x, w, residual=pair[:4], out=pair[1:5])
