"""The expert layer on 16-bit weights where its activation needs all of float32: sums that are known exactly, in float32 too."""

import math

import pytest
import torch

import mlc_llm_amd as gq
from mlc_llm_amd import ops
from test_gpu_dense import close, gated_ref, linear_ref, moe_ref

HALVES = [torch.float16, torch.bfloat16]
pytestmark = pytest.mark.gpu


def _ints(g, most, *shape):
    return torch.randint(-most, most + 1, shape, generator=g).double()


def _pow2(exponents):
    return 2.0 ** torch.as_tensor(exponents, dtype=torch.float64)


# Whole numbers times powers of two.  x has 48 numbers other than 0 in a row, of at most 8, as W13's: a gate or an up value is at most 48 * 64 units, most
# are below 1000, and their product takes up to 23 bits.  Experts of equal logits weigh 1, 1/2 or 1/4.  A row of W2 has four numbers other than 0, so that all sums of
# products stay below 2^24 units (asserted below) and are exact in float32, in any order.  The one rounding is the output's.
def _layer(g, dtype, t, hidden, inter, experts, k, x_exp, gate_exp, up_exp, w2_exp, without=()):
    """x_exp: [t] exponents; gate_exp, up_exp: [inter]; w2_exp: [inter], of the numbers that the columns of W2 hold; without: activations that are 0."""
    x = torch.zeros(t, hidden, dtype=torch.float64)
    count = min(48, hidden)
    at = torch.stack([torch.randperm(hidden, generator=g)[:count] for _ in range(t)])
    x.scatter_(1, at, _ints(g, 8, t, count))
    unit = _pow2(x_exp)[:, None]
    w13 = _ints(g, 8, experts, 2 * inter, hidden)
    w13[:, list(without)] = 0
    w2 = torch.zeros(experts, hidden, inter, dtype=torch.float64)
    # the four columns of a row are of one block of 64, in all experts the same block
    blocks = (inter + 63) // 64
    first = 64 * torch.randint(0, blocks, (1, hidden, 1), generator=g)
    column = (first + torch.randint(0, 64, (experts, hidden, 4), generator=g)).clamp(max=inter - 1)
    sign = 2.0 * torch.randint(0, 2, (experts, hidden, 4), generator=g).double() - 1
    w2.scatter_(2, column, sign)
    logits = torch.full((t, experts), -60.0)
    ids = torch.stack([torch.randperm(experts, generator=g)[:k] for _ in range(t)])
    logits.scatter_(1, ids, 30.0)
    y, size = torch.zeros(t, hidden, dtype=torch.float64), torch.zeros(t, hidden, dtype=torch.float64)
    scale = _pow2(gate_exp) + 0 * _pow2(up_exp)
    for e in range(experts):
        rows = (ids == e).any(1)
        gate, up = (x[rows] @ w13[e].t()).chunk(2, 1)
        h = gate * up
        w = w2[e] * (scale * _pow2(up_exp) * _pow2(w2_exp))
        y[rows] += h @ w.t() / k
        size[rows] += h.abs() @ w2[e].abs().t() / k
    assert size.max() * k < 2**24
    y = y * unit * unit
    w13 = w13 * torch.cat([_pow2(gate_exp), _pow2(up_exp)])[:, None]
    w2 = w2 * _pow2(w2_exp)
    assert y.abs().max() < torch.finfo(dtype).max
    for of in (x * unit, w13, w2):
        assert torch.equal(of.to(dtype).double(), of)
    return ((x * unit).to(dtype).cuda(), logits.cuda(), w13.to(dtype).cuda(), w2.to(dtype).cuda()), y.float().to(dtype).cuda()


# (tokens, hidden, inter, experts, top_k, part of the kernel's note): eight rows a segment through LDS, sixteen and 32 in registers, x kept in the first
# kernel and not, one and several shares
LAYERS = [(1, 2048, 1408, 16, 4, "up to 8 rows"), (1, 64, 72, 4, 1, "up to 8 rows"), (1, 520, 200, 9, 2, "up to 8 rows"), (1, 4104, 2056, 3, 1, "up to 8 rows"),
          (3, 64, 72, 4, 1, "up to 16 rows"), (8, 520, 200, 9, 2, "up to 16 rows"), (16, 1032, 264, 20, 4, "up to 16 rows"), (12, 264, 328, 2, 2, "up to 16 rows"),
          (40, 136, 1032, 6, 2, "up to 16 rows"), (40, 2048, 1024, 8, 2, "up to 16 rows"), (64, 2048, 1032, 4, 2, "up to 32 rows")]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,hidden,inter,experts,k,note", LAYERS)
def test_activation_is_held_in_float32(t, hidden, inter, experts, k, note, dtype):
    """Products of 23 bits that cancel, of sizes that a 16-bit type does not hold or hardly: large and small tokens, magnitudes that rise and fall along K."""
    g = torch.Generator().manual_seed(t + hidden + inter)
    flat, steps = torch.zeros(inter), (torch.arange(inter) // 64).double()
    rise = torch.floor(steps * (12 / max(1.0, steps.max().item())))
    tokens = torch.arange(t) % 5
    if dtype == torch.float16:
        # activations beyond float16's largest number, by 2^2 and 2^8; in units of 2^-40, below its smallest; of many sizes
        scales = [(torch.zeros(t), flat, flat, flat - 12), (torch.zeros(t), flat + 3, flat + 3, flat - 14), (tokens - 10, flat - 10, flat - 10, flat + 12),
                  (torch.zeros(t), rise - 10, flat, -rise + 2), (torch.zeros(t), -rise + 2, flat, rise - 14)]
    else:
        scales = [(torch.zeros(t), flat, flat, flat), (tokens + 40, flat, flat + 10, flat - 60), (tokens - 30, flat - 20, flat - 20, flat + 60),
                  (tokens, rise - 10, flat, -rise + 2), (tokens, -rise + 2, flat, rise - 14)]
    scales.append((*scales[2], [n for n in range(inter) if n // 64 < 9 or n % 64 < 16]))  # small ones behind zeros
    for i, exps in enumerate(scales):
        args, want = _layer(g, dtype, t, hidden, inter, experts, k, *exps)
        got = ops.dense_moe(*args, k, activation=None)
        assert note in gq._lib.last_kernel()
        assert torch.equal(got, want), (i, (got != want).sum().item(), got.numel())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,experts", [(1, 2), (2, 4), (24, 3), (60, 2)])
def test_infinities_of_the_second_product(t, experts, dtype):
    """An infinity among w2's numbers, or an activation beyond float32, gives what the formula gives: an infinity of its sign, and NaN where infinities of
    both signs or an infinity and a zero meet."""
    hidden, inter = 64, 1032
    x = torch.zeros(t, hidden, dtype=dtype, device="cuda")
    x[:, 0], x[:, 1] = 3.0, 1.0
    w13 = torch.zeros(experts, 2 * inter, hidden, dtype=dtype, device="cuda")
    w13[:, :, 0], w13[:, :, 1] = 1 / 3, 2.0**-10  # activations near 1 with many bits
    w2 = torch.ones(experts, hidden, inter, dtype=dtype, device="cuda")
    logits = torch.full((t, experts), -50.0, device="cuda")
    logits[:, 1] = 50.0
    plain = ops.dense_moe(x, logits, w13, w2, 1, activation=None)
    assert plain.isfinite().all()
    w2[1, 1, 5], w2[1, 2, 70], w2[1, 3, 5], w2[1, 3, 6] = math.inf, -math.inf, math.inf, -math.inf
    w2[0] = math.nan  # (nobody's)
    got = ops.dense_moe(x, logits, w13, w2, 1, activation=None)
    assert (got[:, 1] == math.inf).all() and (got[:, 2] == -math.inf).all() and got[:, 3].isnan().all()
    others = [n for n in range(hidden) if n not in (1, 2, 3)]
    assert torch.equal(got[:, others], plain[:, others])
    w2[1] = 0.5
    w2[1, 7], w2[1, 9, 130] = -0.25, 0.0
    if dtype == torch.bfloat16:
        w13[1, 130, 0] = w13[1, inter + 130, 0] = 2.0**100  # 9 * 2^200
    else:
        w13[1, :, 0] = 100.0  # the others 9 * 10^4
        w13[1, 130, 0] = math.inf
    got = ops.dense_moe(x, logits, w13, w2, 1, activation=None)
    others = [n for n in range(hidden) if n not in (7, 9)]
    assert (got[:, 7] == -math.inf).all() and got[:, 9].isnan().all() and (got[:, others] == math.inf).all()


# (rows of x, rows of W, K): tiles of the last round that another form takes, after whole rounds of 256 x 256 and 256 x 160 ones; columns and K that end inside tiles,
# W's rows from which the other form works in the middle of both halves of a gated one
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("m,n,k", [(2048, 9002, 264), (2048, 9008, 520), (1030, 14504, 520), (777, 28674, 520), (2000, 28676, 1032), (200, 66008, 264)])
def test_columns_that_another_form_takes(m, n, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(n + k)
    x, w = (torch.randn(r, k, generator=g, device="cuda") for r in (m, n))
    x, w = x.to(dtype), (w / k**0.5).to(dtype)
    bias = torch.randn(n, generator=g, device="cuda").to(dtype)
    residual = torch.randn(m, n, generator=g, device="cuda").to(dtype)
    close(ops.dense_linear(x, w, bias, "gelu", residual), linear_ref(x, w, bias, "gelu", residual, dtype))
    assert "rows of W from" in gq._lib.last_kernel()
    close(ops.dense_linear(x, w, out_dtype=torch.float32), linear_ref(x, w, None, None, None, torch.float32))
    close(ops.dense_linear_gated(x, w, bias), gated_ref(x, w, bias, "silu", dtype))
    assert "rows of W from" in gq._lib.last_kernel() and "gated" in gq._lib.last_kernel()


@pytest.mark.parametrize("m,n,k", [(2048, 9008, 264), (777, 28680, 520)])
def test_columns_that_another_form_takes_in_a_graph(m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = (torch.randn(r, k, generator=g, device="cuda").to(torch.float16) for r in (m, n))
    ops.dense_linear(x, w), ops.dense_linear_gated(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = ops.dense_linear(x, w, activation="relu"), ops.dense_linear_gated(x, w)
        assert "rows of W from" in gq._lib.last_kernel()
    for _ in range(3):
        x.copy_(torch.randn(m, k, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ops.dense_linear(x, w, activation="relu")) and torch.equal(b, ops.dense_linear_gated(x, w))


# x in registers with four, eight and sixteen experts a lane of the routing, the fullest tables last: 512 experts, 2048 slots
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,hidden,inter,experts,k", [(64, 2048, 1024, 128, 8), (64, 1600, 1032, 200, 8), (64, 3600, 1024, 130, 5), (64, 1544, 1024, 300, 32), (64, 2048, 1024, 512, 32),
                                                      (48, 4096, 1024, 70, 32), (64, 3592, 1024, 257, 9)])
def test_x_in_registers_of_many_experts(t, hidden, inter, experts, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(hidden + experts)
    x = torch.randn(t, hidden, generator=g, device="cuda").to(dtype)
    w13 = torch.empty(experts, 2 * inter, hidden, dtype=dtype, device="cuda")
    w2 = torch.empty(experts, hidden, inter, dtype=dtype, device="cuda")
    for w in (w13, w2):
        for part in w:
            part.copy_(torch.randn(part.shape, generator=g, device="cuda") / part.shape[1] ** 0.5)
    logits = torch.randn(t, experts, generator=g, device="cuda")
    for skewed in (False, True):
        if skewed:  # all tokens to the last experts
            logits[:, -k:] += 20.0
        weights, ids = ops.moe_gating(logits, k)
        got = ops.dense_moe(x, logits, w13, w2, k)
        assert gq._lib.last_kernel().endswith("x kept")
        close(got, moe_ref(x, weights, ids, w13, w2, "silu", dtype))
        assert torch.equal(got, ops.dense_moe(x, logits, w13, w2, k))


def _filled(g, dtype, *shape, scale=1.0):
    """Normal numbers, a part of the rows at a time."""
    w = torch.empty(shape, dtype=dtype, device="cuda")
    for part in w.view(-1, shape[-1]).split(max(1, (1 << 27) // shape[-1])):
        part.copy_(scale * torch.randn(part.shape, generator=g, device="cuda"))
    return w


def _whole(g, dtype, *shape):
    """Whole numbers of at most 8."""
    return _filled(g, dtype, *shape, scale=4.0).clamp_(-8, 8).round_()


def _few(g, dtype, rows, k):
    """Rows of 48 whole numbers of at most 8 among zeros, the last number of a row among them: products with _whole's are exact in float32, in any order."""
    x = torch.zeros(rows, k, dtype=dtype, device="cuda")
    at = torch.randint(0, k, (rows, 48), generator=g, device="cuda")
    at[:, 0] = k - 1
    return x.scatter_(1, at, _whole(g, dtype, rows, 48))


LONGEST = (1 << 23) - 136


@pytest.mark.parametrize("form", [-1, 0, 10])
@pytest.mark.parametrize("m,n", [(1, 24), (7, 40), (12, 24), (60, 72), (300, 280)])
def test_longest_rows(m, n, form):
    """K just below the limit: a tile's offsets come near 2^32 bytes."""
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w = _few(g, torch.bfloat16, m, LONGEST), _whole(g, torch.bfloat16, n, LONGEST)
    want = torch.cat([r[:, r[0] != 0].double() @ w[:, r[0] != 0].double().t() for r in x.split(1)])
    gq._lib.set_option("gemm_variant", form)
    gq._lib.set_option("gemm_split_k", -1 if form < 0 else 1)
    try:
        assert torch.equal(ops.dense_linear(x, w, out_dtype=torch.float32).double(), want)
        got = ops.dense_linear_gated(x, w, activation=None, out_dtype=torch.float32)
        assert torch.equal(got.double(), want[:, : n // 2] * want[:, n // 2 :])
    finally:
        gq._lib.set_option("gemm_variant", -1)
        gq._lib.set_option("gemm_split_k", -1)


@pytest.mark.parametrize("t,hidden,inter,experts,k", [(3, LONGEST, 8, 3, 2), (64, LONGEST, 8, 2, 1), (5, 8, LONGEST, 3, 2), (64, 16, LONGEST, 2, 1)])
def test_longest_rows_of_an_expert_layer(t, hidden, inter, experts, k):
    g = torch.Generator(device="cuda").manual_seed(t)
    dtype = torch.bfloat16
    x = _few(g, dtype, t, hidden) if hidden > 48 else _whole(g, dtype, t, hidden)
    w13 = _whole(g, dtype, experts, 2 * inter, hidden)
    w2 = torch.zeros(experts, hidden, inter, dtype=dtype, device="cuda")  # two numbers other than 0 in a row, one of them in its last eight
    w2.scatter_(2, torch.randint(0, inter, (experts, hidden, 1), generator=g, device="cuda"), 1.0)
    w2.scatter_(2, torch.randint(inter - 8, inter, (experts, hidden, 1), generator=g, device="cuda"), -1.0)
    logits = torch.full((t, experts), -60.0, device="cuda")
    ids = torch.stack([torch.randperm(experts, generator=g, device="cuda")[:k] for _ in range(t)])
    logits.scatter_(1, ids, 30.0)
    want = torch.zeros(t, hidden, dtype=torch.float64, device="cuda")
    for e in range(experts):
        rows = (ids == e).any(1)
        some = x[rows].ne(0).any(0)
        gate, up = (x[rows][:, some].double() @ w13[e][:, some].double().t()).chunk(2, 1)
        used = w2[e].ne(0).any(0)
        want[rows] += (gate * up)[:, used] @ w2[e][:, used].double().t() / k
    got = ops.dense_moe(x, logits, w13, w2, k, activation=None)
    assert torch.equal(got, want.float().to(dtype))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,hidden,inter,experts,k", [(1, 256, 128, 8, 2), (16, 2048, 768, 16, 4), (64, 2048, 1024, 4, 2)])
def test_output_of_an_expert_layer_in_place_of_x(t, hidden, inter, experts, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(hidden)
    x, logits = _filled(g, dtype, t, hidden), torch.randn(t, experts, generator=g, device="cuda")
    w13, w2 = _filled(g, dtype, experts, 2 * inter, hidden, scale=hidden**-0.5), _filled(g, dtype, experts, hidden, inter, scale=inter**-0.5)
    want = ops.dense_moe(x, logits, w13, w2, k)
    size = gq._lib.lib().mi355gq_dense_moe_workspace_bytes(t, hidden, inter, experts, k)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    gq._lib.call("mi355gq_dense_moe", x.data_ptr(), logits.data_ptr(), None, t, hidden, inter, experts, k, 0, 1, 1, 1, 1.0, ops._MODEL_DTYPES[logits.dtype],
                 w13.data_ptr(), w2.data_ptr(), ops._activation("silu"), ops._MODEL_DTYPES[dtype], x.data_ptr(), ws.data_ptr(), size, ops._stream())
    assert torch.equal(x, want)


def test_two_expert_layers_at_once():
    """Calls of two streams, each with scratch of its own."""
    g = torch.Generator(device="cuda").manual_seed(8)
    layers = []
    for t, hidden, inter, experts, k, dtype in ((9, 1024, 776, 24, 3, torch.float16), (64, 2048, 1024, 8, 2, torch.bfloat16)):
        args = [_filled(g, dtype, t, hidden), torch.randn(t, experts, generator=g, device="cuda"), _filled(g, dtype, experts, 2 * inter, hidden, scale=hidden**-0.5),
                _filled(g, dtype, experts, hidden, inter, scale=inter**-0.5), k]
        layers.append((args, ops.dense_moe(*args), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (args, _, stream) in enumerate(layers):
            with torch.cuda.stream(stream):
                got[i].append(ops.dense_moe(*args))
    torch.cuda.synchronize()
    for i, (_, want, _) in enumerate(layers):
        assert all(torch.equal(y, want) for y in got[i])
