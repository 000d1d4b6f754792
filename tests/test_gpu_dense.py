"""Operators on 16-bit weights against their definitions in float64, within bounds that follow from their roundings.

A sum of K products in float32, in any order, is off by at most K 2^-23 of the sum of their magnitudes (K - 1 additions of 2^-24 each,
and as much again for a matrix unit that truncates).  Behind it an activation passes an error on at most 1.13 times (the steepest slope
of gelu and silu) and is itself good to 1e-6 of its value; a rounding is off by half a step."""

import math

import pytest
import torch

import mlc_llm_amd as gq
from mlc_llm_amd import ops

HALVES = [torch.float16, torch.bfloat16]
UNIT = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-149}  # half a step of the smallest numbers
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]
pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _normal(g, dtype, *shape, scale=1.0):
    return (scale * torch.randn(*shape, generator=g)).to(dtype).cuda()


def act_of(v, name):
    if name == "relu":
        return v.clamp(min=0)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * torch.erfc(-(0.5**0.5) * v)  # = v Phi(v), with all digits of its tail
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3))  # = v / 2 (1 + tanh(half of that))
    return v


def product(x, w, bias=None):
    """(y, error bound) of x w^T + bias in float32."""
    x, w = x.double(), w.double()
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, (x.shape[1] + 2) * 2.0**-23 * size


def rounded(err, y, dtype):
    return err + UNIT[dtype] * (y.abs() + err) + TINY[dtype]


def linear_ref(x, w, bias, act, residual, out_dtype):
    v, err = product(x, w, bias)
    y = act_of(v, act)
    if act:
        err = 1.13 * err + 1e-6 * y.abs() + 1e-37
    if residual is not None:
        y = y + residual.double()
        err = err + 2.0**-23 * (y.abs() + residual.double().abs())
    return y, rounded(err, y, out_dtype)


def gated_ref(x, w, bias, act, out_dtype):
    v, err = product(x, w, bias)
    (g, u), (eg, eu) = v.chunk(2, 1), err.chunk(2, 1)
    a = act_of(g, act)
    if act:
        eg = 1.13 * eg + 1e-6 * a.abs() + 1e-37
    y = a * u
    err = eg * u.abs() + a.abs() * eu + eg * eu + 2.0**-23 * y.abs()
    return y, rounded(err, y, out_dtype)


def close(got, want):
    y, bound = want
    assert got.shape == y.shape
    worst = ((got.double() - y).abs() / bound).max().item() if y.numel() else 0.0
    assert worst <= 1.0, f"{worst} of the bound ({gq._lib.last_kernel()})"


# (rows, columns, K): one of everything, tiles that end inside, every kernel's range of rows
SIZES = [(1, 1, 1), (1, 16, 8), (2, 17, 40), (3, 5, 33), (1, 4096, 4096), (5, 8, 14336), (7, 515, 136), (16, 128, 2048), (17, 130, 264),
         (33, 64, 72), (48, 512, 1408), (63, 1000, 8), (64, 96, 4096), (65, 257, 1000), (129, 515, 136), (200, 72, 2056), (257, 128, 64),
         (300, 1000, 520), (513, 769, 392), (1030, 264, 328)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(m, n, k, dtype):
    g = _gen(m * 7 + n * 3 + k)
    x, w = _normal(g, dtype, m, k), _normal(g, dtype, n, k, scale=k**-0.5)
    bias, residual = _normal(g, dtype, n), _normal(g, dtype, m, n)
    close(ops.dense_linear(x, w), linear_ref(x, w, None, None, None, dtype))
    for i, act in enumerate(ACTS):
        out_dtype = torch.float32 if i % 2 else dtype
        b, r = (bias if i != 2 else None), (residual if i != 3 else None)
        got = ops.dense_linear(x, w, bias=b, activation=act, residual=r, out_dtype=out_dtype)
        assert got.dtype == out_dtype
        close(got, linear_ref(x, w, b, act, r, out_dtype))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gated(m, n, k, dtype):
    g = _gen(m * 5 + n * 11 + k)
    x, w, bias = _normal(g, dtype, m, k), _normal(g, dtype, 2 * n, k, scale=k**-0.5), _normal(g, dtype, 2 * n)
    close(ops.dense_linear_gated(x, w), gated_ref(x, w, None, "silu", dtype))
    for i, act in enumerate(ACTS):
        out_dtype = torch.float32 if i % 2 else dtype
        b = bias if i != 2 else None
        close(ops.dense_linear_gated(x, w, bias=b, activation=act, out_dtype=out_dtype), gated_ref(x, w, b, act, out_dtype))


@pytest.mark.parametrize("m,n,k", [(1, 9728, 2560), (8, 4872, 2600), (3, 8200, 2888), (16, 4868, 2600), (2, 100, 5000)])
def test_blocks_of_a_wave_past_its_ring(m, n, k):
    """K of five to eleven blocks a wave, over several items each."""
    g = _gen(n + k)
    for dtype in HALVES:
        x, w, bias = _normal(g, dtype, m, k), _normal(g, dtype, n, k, scale=k**-0.5), _normal(g, dtype, n)
        close(ops.dense_linear(x, w, bias=bias, activation="silu"), linear_ref(x, w, bias, "silu", None, dtype))
        assert "dense_rows" in gq._lib.last_kernel()
        close(ops.dense_linear_gated(x, w), gated_ref(x, w, None, "silu", dtype))


@pytest.mark.parametrize("shares", [1, 3])
@pytest.mark.parametrize("form", range(11))
def test_tile_forms(form, shares):
    """Every tile form, whole and in shares of K, on tiles that end inside in all directions."""
    g = _gen(form * 10 + shares)
    gq._lib.set_option("gemm_variant", form)
    gq._lib.set_option("gemm_split_k", shares)
    try:
        for i, (m, n, k) in enumerate([(17, 40, 776), (33, 257, 1032), (160, 130, 776), (200, 520, 776), (300, 129, 968), (521, 392, 1288)]):
            dtype = HALVES[i % 2]
            x, w, bias = _normal(g, dtype, m, k), _normal(g, dtype, n, k, scale=k**-0.5), _normal(g, dtype, n)
            r = _normal(g, dtype, m, n)
            got = ops.dense_linear(x, w, bias=bias, activation="gelu", residual=r)
            assert f"{shares} shares" in gq._lib.last_kernel()
            close(got, linear_ref(x, w, bias, "gelu", r, dtype))
            x, w, bias = _normal(g, dtype, m, k), _normal(g, dtype, 2 * n, k, scale=k**-0.5), _normal(g, dtype, 2 * n)
            close(ops.dense_linear_gated(x, w, bias=bias), gated_ref(x, w, bias, "silu", dtype))
    finally:
        gq._lib.set_option("gemm_variant", -1)
        gq._lib.set_option("gemm_split_k", -1)


@pytest.mark.parametrize("m,n,k", [(2048, 14500, 520), (300, 30000, 264)])
def test_rest_of_the_last_round(m, n, k):
    """More tiles than run at a time: columns in one form, the rest of them in another."""
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, k, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(n, k, generator=g, device="cuda") / k**0.5).to(torch.bfloat16)
    close(ops.dense_linear(x, w, activation="silu"), linear_ref(x, w, None, "silu", None, torch.bfloat16))
    close(ops.dense_linear_gated(x, w), gated_ref(x, w, None, "silu", torch.bfloat16))


@pytest.mark.parametrize("m", [1, 6, 20, 40, 130])
def test_unaligned_pointers_and_leading_dimensions(m):
    """Tensors in the middle of others, at 2 bytes, and x of more than two dimensions."""
    g = _gen(m)
    dtype = torch.bfloat16
    k, n = 264, 136

    def inside(*shape):
        size = math.prod(shape)
        return _normal(g, dtype, size + 9)[1 : 1 + size].view(shape)

    x, w, b, r = inside(m, k), inside(n, k), inside(n), inside(m, n)
    for xx in (x, x.clone()):
        for ww in (w, w.clone()):
            for bb, rr in ((b, r), (b.clone(), r.clone()), (None, r)):
                close(ops.dense_linear(xx, ww, bias=bb, activation="silu", residual=rr), linear_ref(xx, ww, bb, "silu", rr, dtype))
            close(ops.dense_linear_gated(xx, ww, bias=b, activation="gelu"), gated_ref(xx, ww, b, "gelu", dtype))
    out = torch.full((m * n + 9,), 7.0, dtype=dtype, device="cuda")
    ops.dense_linear(x, w, out=out[3 : 3 + m * n].view(m, n))
    close(out[3 : 3 + m * n].view(m, n), linear_ref(x, w, None, None, None, dtype))
    assert (out[:3] == 7).all() and (out[3 + m * n :] == 7).all()
    y = ops.dense_linear(x.view(m, 1, 1, k), w)
    assert y.shape == (m, 1, 1, n) and torch.equal(y.view(m, n), ops.dense_linear(x, w))
    one = ops.dense_linear(x[0].clone(), w)
    assert one.shape == (n,)


@pytest.mark.parametrize("m", [1, 9, 33, 150])
def test_in_place_residual_and_neighbours(m):
    g = _gen(m + 50)
    n, k = 520, 1032
    x, w = _normal(g, torch.float16, m, k), _normal(g, torch.float16, n, k, scale=k**-0.5)
    wide = torch.full((m + 2, n), -3.0, dtype=torch.float16, device="cuda")
    hidden = wide[1 : m + 1]
    hidden.copy_(_normal(g, torch.float16, m, n))
    want = linear_ref(x, w, None, "gelu_tanh", hidden.clone(), torch.float16)
    assert ops.dense_linear(x, w, activation="gelu_tanh", residual=hidden, out=hidden).data_ptr() == hidden.data_ptr()
    close(hidden, want)
    assert (wide[0] == -3).all() and (wide[m + 1] == -3).all()


@pytest.mark.parametrize("m", [1, 20, 100])
def test_empty(m):
    w = torch.zeros(0, 64, dtype=torch.float16, device="cuda")
    assert ops.dense_linear(torch.ones(m, 64, dtype=torch.float16, device="cuda"), w).shape == (m, 0)
    assert ops.dense_linear_gated(torch.ones(m, 64, dtype=torch.float16, device="cuda"), w).shape == (m, 0)
    w = torch.zeros(m, 64, dtype=torch.float16, device="cuda")
    assert ops.dense_linear(torch.ones(0, 64, dtype=torch.float16, device="cuda"), w).shape == (0, m)
    assert ops.dense_linear_gated(torch.ones(2, 0, 64, dtype=torch.float16, device="cuda"), torch.cat([w, w])).shape == (2, 0, m)


def test_activations_over_their_range():
    """W = 1, x = v: the activation of every float16 number, in float32."""
    v = torch.arange(-(2**15), 2**15, dtype=torch.int32).to(torch.int16).view(torch.float16).cuda()
    v = v[v.isfinite()]
    x = torch.zeros(len(v), 8, dtype=torch.float16, device="cuda")
    x[:, 0] = v
    w = torch.ones(8, 8, dtype=torch.float16, device="cuda")
    for act in ACTS[1:]:
        want = act_of(v.double(), act)
        # (an activation far out on the negative side may end below float32's smallest number, and its factors do a little before)
        bound = 2e-6 * want.abs() + 1e-36 * v.double().abs() + 1e-37
        if act == "gelu":  # exp(-v^2 / 2) from v^2 in float32
            bound = bound + want.abs() * v.double() ** 2 * 2.0**-23
        if act in ("gelu_tanh", "silu"):  # the exponent in float32, likewise
            e = v.double().abs() if act == "silu" else 1.6 * (v.double().abs() + 0.044715 * v.double().abs() ** 3)
            bound = bound + want.abs() * e * 2.0**-21
        got = ops.dense_linear(x, w, activation=act, out_dtype=torch.float32)[:, 0].double()
        assert ((got - want).abs() <= bound).all(), act


def test_not_finite():
    inf, nan = math.inf, math.nan
    for m in (2, 20, 100):
        x = torch.ones(m, 64, dtype=torch.float16, device="cuda")
        w = torch.zeros(24, 64, dtype=torch.float16, device="cuda")
        w[:, 0] = 1
        w[3, 5], w[4, 5], w[5, 5] = inf, -inf, nan
        y = ops.dense_linear(x, w)
        assert (y[:, 3] == inf).all() and (y[:, 4] == -inf).all() and y[:, 5].isnan().all()
        assert y[:, [i for i in range(24) if i not in (3, 4, 5)]].eq(1).all()
        for act in ACTS[1:]:
            y = ops.dense_linear(x, w, activation=act)
            assert (y[:, 3] == inf).all() and y[:, 5].isnan().all(), act
            assert (y[:, 4] == 0).all() if act == "relu" else y[:, 4].isnan().all(), act
        x[1, 7] = nan  # one token's trouble is its own
        y = ops.dense_linear(x, w)
        assert y[1].isnan().all() and y[0, 0] == 1


@pytest.mark.parametrize("m", [2, 12, 30, 100, 300])
def test_not_finite_in_the_next_row(m):
    """Rows that end inside a block of K: what stands behind them, the next row's first numbers, is not theirs."""
    g = _gen(m)
    k, n = 200, 81
    x, w = _normal(g, torch.bfloat16, m, k), _normal(g, torch.bfloat16, n, k, scale=k**-0.5)
    clean, clean_gated = ops.dense_linear(x, w), ops.dense_linear_gated(x, w[:80])
    w[1::2], x[1::2] = math.nan, math.inf
    got = ops.dense_linear(x, w)
    assert torch.equal(got[::2, ::2], clean[::2, ::2])
    assert got[:, 1::2].isnan().all()
    assert torch.equal(ops.dense_linear_gated(x, w[:80])[::2, ::2], clean_gated[::2, ::2])


def test_more_rows_than_a_launch_takes():
    m, n, k = (1 << 20) + 77, 24, 40
    g = torch.Generator(device="cuda").manual_seed(4)
    x, w = (torch.randn(r, k, generator=g, device="cuda").to(torch.float16) for r in (m, n))
    r = torch.randn(m, n, generator=g, device="cuda").to(torch.float16)
    y = ops.dense_linear(x, w, activation="relu", residual=r, out_dtype=torch.float32)
    rows = torch.tensor([0, 1, (1 << 20) - 1, 1 << 20, (1 << 20) + 1, m - 1], device="cuda")
    close(y[rows], linear_ref(x[rows], w, None, "relu", r[rows], torch.float32))
    close(ops.dense_linear_gated(x, w)[rows], gated_ref(x[rows], w, None, "silu", torch.float16))


@pytest.mark.parametrize("m", [3, 40])
def test_weights_beyond_4_gib(m):
    n, k = 270000, 8192
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.empty(n, k, dtype=torch.bfloat16, device="cuda")
    for part in w.split(30000):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") / 90)
    x = torch.randn(m, k, generator=g, device="cuda").to(torch.bfloat16)
    rows = torch.tensor([0, 1, 131071, 131072, 131073, 262143, 262144, 262145, n // 2 - 1, n // 2, n - 17, n - 1], device="cuda")
    y = ops.dense_linear(x, w)
    close(y[:, rows], linear_ref(x, w[rows], None, None, None, torch.bfloat16))
    y = ops.dense_linear_gated(x, w)
    rows = torch.tensor([0, 1, 17, 65535, 65536, 131071, 131072, 134999], device="cuda")
    close(y[:, rows], gated_ref(x, torch.cat([w[rows], w[rows + n // 2]]), None, "silu", torch.bfloat16))


def test_results_beyond_2_to_the_31():
    m, n, k = 70001, 32776, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w = (torch.randn(r, k, generator=g, device="cuda").to(torch.float16) for r in (m, n))
    y = ops.dense_linear(x, w, activation="relu")
    rows = torch.tensor([0, 1, 255, 256, 65535, 65536, 65537, m - 2, m - 1], device="cuda")
    close(y[rows], linear_ref(x[rows], w, None, "relu", None, torch.float16))


@pytest.mark.parametrize("m", [1, 12, 40, 300])
def test_graph_replays(m):
    g = _gen(m)
    k, n = 1024, 520
    x, w, r = _normal(g, torch.bfloat16, m, k), _normal(g, torch.bfloat16, n, k, scale=k**-0.5), _normal(g, torch.bfloat16, m, n)
    ops.dense_linear(x, w, residual=r), ops.dense_linear_gated(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = ops.dense_linear(x, w, activation="silu", residual=r), ops.dense_linear_gated(x, w, activation="gelu")
    for i in range(4):
        x.copy_(_normal(g, torch.bfloat16, m, k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ops.dense_linear(x, w, activation="silu", residual=r))
        assert torch.equal(b, ops.dense_linear_gated(x, w, activation="gelu"))


def test_other_stream():
    g = _gen(3)
    w = _normal(g, torch.float16, 2048, 2048, scale=2048**-0.5)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        x = torch.ones(64, 2048, dtype=torch.float16, device="cuda")
        for _ in range(20):
            x = ops.dense_linear(x, w, activation="silu")
        y = x * 2
    side.synchronize()
    z = torch.ones(64, 2048, dtype=torch.float16, device="cuda")
    for _ in range(20):
        z = ops.dense_linear(z, w, activation="silu")
    assert torch.equal(y, z * 2)


# ---- the expert layer ----


def moe_ref(x, weights, ids, w13, w2, act, dtype):
    """(y, bound) of a layer on routed tokens, in float64 from the very weights and ids of moe_gating."""
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    err = torch.zeros_like(y)
    for e in ids.unique().tolist():
        token, slot = torch.nonzero(ids == e, as_tuple=True)
        v, ev = product(x[token], w13[e])
        (g, u), (eg, eu) = v.chunk(2, 1), ev.chunk(2, 1)
        a = act_of(g, act)
        if act:
            eg = 1.13 * eg + 1e-6 * a.abs() + 1e-37
        w = weights[token, slot].double()[:, None]
        h = w * a * u
        # the float32 product; held as two numbers, half a step of a half step, or of the smallest numbers
        eh = w.abs() * (eg * u.abs() + a.abs() * eu + eg * eu) + (2.0**-23 + UNIT[dtype] ** 2) * h.abs() + 2 * TINY[dtype]
        d, ed = product(h, w2[e])
        y[token] += d
        # a sum over twice as many products, and over the token's experts
        err[token] += 2 * ed + eh @ w2[e].double().abs().t() + ids.shape[1] * 2.0**-23 * (h.abs() @ w2[e].double().abs().t())
    return y, rounded(err, y, dtype)


def _layer(g, dtype, t, hidden, inter, experts, logits_dtype=torch.float32):
    return (_normal(g, dtype, t, hidden), _normal(g, logits_dtype, t, experts, scale=1.5), _normal(g, dtype, experts, 2 * inter, hidden, scale=hidden**-0.5),
            _normal(g, dtype, experts, hidden, inter, scale=inter**-0.5))


# (tokens, hidden, inter, experts, top_k): each number of experts a lane holds, shares of the second product, sizes that end inside a block
LAYERS = [(1, 256, 128, 8, 2), (1, 2048, 1408, 64, 6), (2, 64, 8, 4, 4), (3, 72, 200, 5, 1), (4, 512, 1032, 8, 2), (7, 8, 8, 1, 1), (15, 520, 136, 60, 8),
          (16, 2048, 768, 128, 8), (17, 264, 328, 24, 3), (31, 136, 264, 160, 6), (32, 1024, 512, 16, 4), (33, 104, 64, 300, 32), (50, 256, 96, 512, 8),
          (64, 512, 264, 8, 2), (64, 136, 72, 2, 2), (64, 64, 64, 64, 32)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,hidden,inter,experts,k", LAYERS)
def test_moe(t, hidden, inter, experts, k, dtype):
    g = _gen(t * 31 + hidden + inter + experts)
    for i, (scoring, act, logits_dtype) in enumerate([("softmax", "silu", torch.float32), ("sigmoid", "gelu_tanh", dtype), ("softmax", "gelu", torch.float32)]):
        x, logits, w13, w2 = _layer(g, dtype, t, hidden, inter, experts, logits_dtype)
        how = {"scoring": scoring, "renormalize": i != 1, "scale": 2.5 if i == 1 else 1.0}
        if i == 1:
            how["bias"] = _normal(g, torch.float32, experts, scale=0.1)
        if i and experts % 4 == 0 and experts // 2 >= k:
            how.update(num_groups=4, top_groups=2)
        weights, ids = ops.moe_gating(logits, k, **how)
        got = ops.dense_moe(x, logits, w13, w2, k, activation=act, **how)
        assert got.dtype == dtype
        close(got, moe_ref(x, weights, ids, w13, w2, act, dtype))
        assert torch.equal(got, ops.dense_moe(x, logits, w13, w2, k, activation=act, **how))


@pytest.mark.parametrize("t", [5, 20, 64])
def test_moe_skewed_routing(t):
    """Every token to the same experts, and one expert of many for all."""
    g = _gen(t)
    x, logits, w13, w2 = _layer(g, torch.bfloat16, t, 256, 200, 40)
    logits[:, 7] = 9.0
    logits[:, 39] = 8.0
    for k in (1, 2, 3):
        weights, ids = ops.moe_gating(logits, k)
        close(ops.dense_moe(x, logits, w13, w2, k), moe_ref(x, weights, ids, w13, w2, "silu", torch.bfloat16))
    logits[:] = 0  # ties: the lowest experts
    weights, ids = ops.moe_gating(logits, 4)
    assert (ids == torch.arange(4, device="cuda")).all()
    close(ops.dense_moe(x, logits, w13, w2, 4), moe_ref(x, weights, ids, w13, w2, "silu", torch.bfloat16))


# x in registers: four, seven and eight blocks of K a wave, K that ends inside a block; segments of 32 rows in the first kernel, of 8 or 16 in the second
KEPT = [(64, 2048, 1024, 4, 2), (33, 1544, 1032, 3, 1), (40, 4096, 1024, 2, 2), (8, 3592, 1024, 4, 2), (64, 2000, 1096, 8, 8), (7, 3584, 1032, 1, 1), (64, 1600, 1024, 60, 3)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,hidden,inter,experts,k", KEPT)
def test_moe_x_in_registers(t, hidden, inter, experts, k, dtype):
    g = _gen(t + hidden + inter)
    x, logits, w13, w2 = _layer(g, dtype, t, hidden, inter, experts)
    for skewed in (False, True):
        if skewed:  # all tokens to the same experts, the last among them
            logits[:, -k:] += 20.0
        weights, ids = ops.moe_gating(logits, k)
        got = ops.dense_moe(x, logits, w13, w2, k)
        assert gq._lib.last_kernel().endswith("x kept")
        close(got, moe_ref(x, weights, ids, w13, w2, "silu", dtype))
        assert torch.equal(got, ops.dense_moe(x, logits, w13, w2, k))
    if experts > k:  # what others chose, or nobody, stays away from a token
        logits[:, 0], logits[0, 0] = -50.0, 60.0
        weights, ids = ops.moe_gating(logits, k)
        want = ops.dense_moe(x, logits, w13, w2, k)
        w13[0, 0] = math.inf
        got = ops.dense_moe(x, logits, w13, w2, k)
        assert not got[0].isfinite().all() and torch.equal(got[1:], want[1:])


@pytest.mark.parametrize("t", [2, 40])
def test_moe_troubles_stay_where_they_are(t):
    """Experts that nobody chose, and those that others chose, may hold anything; a token's NaN is its own."""
    g = _gen(t)
    x, logits, w13, w2 = _layer(g, torch.float16, t, 128, 64, 8)
    logits[:, 3] = -50.0
    logits[0, 5], logits[1:, 5] = 20.0, -40.0  # expert 5: token 0 alone
    weights, ids = ops.moe_gating(logits, 2)
    assert (ids[0] == 5).any() and not (ids[1:] == 5).any() and not (ids == 3).any()
    w13[3], w2[3] = math.nan, math.inf
    w13[5, 0], w2[5, 1] = math.inf, math.nan
    got = ops.dense_moe(x, logits, w13, w2, 2)
    assert got[0, 1].isnan()
    y, bound = moe_ref(x[1:], weights[1:], ids[1:], w13, w2, "silu", torch.float16)
    close(got[1:], (y, bound))
    x[1, 3] = math.nan
    again = ops.dense_moe(x, logits, w13, w2, 2)
    assert again[1].isnan().all() and torch.equal(again[2:], got[2:])


def test_moe_weights_beyond_4_gib():
    t, hidden, inter, experts, k = 12, 4096, 8200, 40, 3
    g = torch.Generator(device="cuda").manual_seed(5)
    w13 = torch.empty(experts, 2 * inter, hidden, dtype=torch.bfloat16, device="cuda")
    w2 = torch.empty(experts, hidden, inter, dtype=torch.bfloat16, device="cuda")
    for w in (w13, w2):
        for part in w:
            part.copy_(torch.randn(part.shape, generator=g, device="cuda") / 80)
    x = torch.randn(t, hidden, generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.randn(t, experts, generator=g, device="cuda")
    logits[0, 39] = logits[1, 0] = 20.0
    weights, ids = ops.moe_gating(logits, k)
    close(ops.dense_moe(x, logits, w13, w2, k), moe_ref(x, weights, ids, w13, w2, "silu", torch.bfloat16))


@pytest.mark.parametrize("t", [1, 16, 40])
def test_moe_graph_replays(t):
    """Two captured layers that take their scratch from one pool, replayed in turn with other work between."""
    g = _gen(t)
    x, logits, w13, w2 = _layer(g, torch.bfloat16, t, 512, 264, 24)
    ops.dense_moe(x, logits, w13, w2, 3)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in (3, 6):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(ops.dense_moe(x, logits, w13, w2, k))
        graphs.append(graph)
    for i in range(4):
        x.copy_(_normal(g, torch.bfloat16, *x.shape))
        logits.copy_(_normal(g, torch.float32, *logits.shape))
        for k, graph, out in zip((3, 6), graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.dense_moe(x, logits, w13, w2, k))


def test_moe_graph_replays_with_x_in_registers():
    g = _gen(77)
    x, logits, w13, w2 = _layer(g, torch.float16, 64, 2048, 1024, 4)
    ops.dense_moe(x, logits, w13, w2, 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.dense_moe(x, logits, w13, w2, 2)
    for i in range(4):
        x.copy_(_normal(g, torch.float16, *x.shape))
        logits.copy_(_normal(g, torch.float32, *logits.shape, scale=0.1 + 3 * i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.dense_moe(x, logits, w13, w2, 2))


# (tokens, hidden, inter, experts, top_k): one token, shares of the second product, 32 columns a workgroup, x in registers with segments of 16 and 32 rows
@pytest.mark.parametrize("t,hidden,inter,experts,k", [(1, 2048, 1408, 64, 6), (16, 2048, 768, 128, 8), (33, 104, 64, 300, 32), (40, 264, 136, 8, 3),
                                                      (40, 2048, 1024, 8, 2), (64, 2048, 1032, 4, 2)])
def test_moe_whatever_its_workspace_holds(t, hidden, inter, experts, k):
    """Scratch full of ones or of an earlier call's, guards behind it and the output, NaN and infinite logits."""
    g = _gen(t + inter)
    x, logits, w13, w2 = _layer(g, torch.bfloat16, t, hidden, inter, experts)
    logits[0] = math.nan
    logits[t // 2, : experts // 2] = math.inf
    logits[t - 1] = -math.inf
    want = ops.dense_moe(x, logits, w13, w2, k)
    weights, ids = ops.moe_gating(logits, k)
    assert ((ids >= 0) & (ids < experts)).all() and all(len(set(row)) == k for row in ids.tolist())
    close(want, moe_ref(x, weights, ids, w13, w2, "silu", torch.bfloat16))
    size = gq._lib.lib().mi355gq_dense_moe_workspace_bytes(t, hidden, inter, experts, k)
    ws = torch.full((size + 256,), 255, dtype=torch.uint8, device="cuda")
    out = torch.full((t * hidden + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    for _ in range(3):
        gq._lib.call("mi355gq_dense_moe", x.data_ptr(), logits.data_ptr(), None, t, hidden, inter, experts, k, 0, 1, 1, 1, 1.0, ops._MODEL_DTYPES[logits.dtype],
                     w13.data_ptr(), w2.data_ptr(), ops._activation("silu"), ops._MODEL_DTYPES[x.dtype], out.data_ptr(), ws.data_ptr(), size, ops._stream())
        assert torch.equal(out[: t * hidden].view(t, hidden), want)
        assert (ws[size:] == 255).all() and (out[t * hidden :] == 7).all()
        out[: t * hidden] = math.nan


def test_router_layer_and_residual_together():
    """As a decoder layer runs them: router logits in float32, experts, a shared gated MLP whose down projection adds the rest up."""
    g = _gen(9)
    dtype, t, hidden, inter, experts, k = torch.bfloat16, 11, 512, 264, 24, 3
    x, _, w13, w2 = _layer(g, dtype, t, hidden, inter, experts)
    router = _normal(g, dtype, experts, hidden, scale=hidden**-0.5)
    up, down = _normal(g, dtype, 2 * inter, hidden, scale=hidden**-0.5), _normal(g, dtype, hidden, inter, scale=inter**-0.5)
    logits = ops.dense_linear(x, router, out_dtype=torch.float32)
    close(logits, linear_ref(x, router, None, None, None, torch.float32))
    routed = ops.dense_moe(x, logits, w13, w2, k)
    weights, ids = ops.moe_gating(logits, k)
    close(routed, moe_ref(x, weights, ids, w13, w2, "silu", dtype))
    shared = ops.dense_linear_gated(x, up, activation="gelu_tanh")
    close(shared, gated_ref(x, up, None, "gelu_tanh", dtype))
    y = ops.dense_linear(shared, down, residual=routed, out=routed)
    assert y.data_ptr() == routed.data_ptr()
    close(y, linear_ref(shared, down, None, None, ops.dense_moe(x, logits, w13, w2, k), dtype))


def test_moe_refuses_more_tokens():
    x, logits, w13, w2 = _layer(_gen(1), torch.float16, 65, 64, 32, 4)
    with pytest.raises(gq._lib.Mi355gqError) as err:
        ops.dense_moe(x, logits, w13, w2, 2)
    assert err.value.code == gq._lib.ERR_UNSUPPORTED and "64 tokens at most" in err.value.message
    assert ops.dense_moe(x[:0], logits[:0], w13, w2, 2).shape == (0, 64)


class Plain(torch.Tensor):
    """A subclass: the native call path declines it, the Python route takes it."""


@pytest.mark.parametrize("lead", [(1,), (2, 3), (40,), ()])
def test_native_and_python_routes_agree(lead):
    g, dtype, n, k = _gen(7), torch.bfloat16, 72, 136
    x, w, b, r = _normal(g, dtype, *lead, k), _normal(g, dtype, n, k), _normal(g, dtype, n), _normal(g, dtype, *lead, n)
    native = gq._lib.native()
    for bias in (None, b):
        for act in ACTS:
            for out_dtype in (None, torch.float32):
                for residual in (None, r):
                    assert isinstance(native.dense_linear(x, w, bias, act, out_dtype, residual, None), torch.Tensor)
                    got = ops.dense_linear(x, w, bias, act, residual, out_dtype)
                    want = ops.dense_linear(x.as_subclass(Plain), w, bias, act, residual, out_dtype)
                    assert got.dtype == want.dtype and got.shape == (*lead, n) and torch.equal(got, want.as_subclass(torch.Tensor))
                    out = torch.empty_like(got)
                    assert native.dense_linear(x, w, bias, act, out_dtype, residual, out) is not None
                    assert ops.dense_linear(x, w, bias, act, residual, out_dtype, out).data_ptr() == out.data_ptr() and torch.equal(out, got)
                assert isinstance(native.dense_linear_gated(x, w, bias, act, out_dtype), torch.Tensor)
                got, want = ops.dense_linear_gated(x, w, bias, act, out_dtype), ops.dense_linear_gated(x.as_subclass(Plain), w, bias, act, out_dtype)
                assert got.dtype == want.dtype and got.shape == (*lead, n // 2) and torch.equal(got, want.as_subclass(torch.Tensor))
    x, logits, w13, w2 = _layer(g, dtype, 5, 128, 64, 8, torch.float16)
    bias = torch.randn(8, device="cuda")
    for how in ({}, {"scoring": "sigmoid", "bias": bias, "num_groups": 2, "top_groups": 1, "renormalize": False, "scale": 2.5, "activation": "gelu"}):
        got, want = ops.dense_moe(x, logits, w13, w2, 2, **how), ops.dense_moe(x.as_subclass(Plain), logits, w13, w2, 2, **how)
        assert torch.equal(got, want.as_subclass(torch.Tensor))
    assert isinstance(native.dense_moe(x, w13, w2, "silu", logits, 2, "softmax", None, 1, 1, True, 1.0), torch.Tensor)
