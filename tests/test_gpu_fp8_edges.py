"""8-bit block-scaled operators where one form ends and another begins: one token beyond the one-row kernel, rows that lie in a wider
buffer, segments of several passes, a layer whose every sum is known exactly, layers that are copied, moved and cast."""

import copy

import pytest
import torch

from mlc_llm_amd import _lib, nn as layers, ops
from test_gpu_fp8 import DTYPES, E4M3, UNIT, _gen, _linear_bound, _step_bound, _weights, block_values, quantized

pytestmark = pytest.mark.gpu


class ExactLayer:
    """An expert layer on whole numbers: gate and up sums below 2^24 are the same in any order, so the activation's bytes are known
    and what remains is the second product, the weighted sum and one rounding."""

    def __init__(self, t, hidden, inter, ne, ids, dtype, top=8):
        g = torch.Generator(device="cuda").manual_seed(t + hidden + inter)

        def whole(*shape):
            return torch.randint(-top, top + 1, shape, generator=g, device="cuda", dtype=torch.int8).to(dtype).float()

        assert top * top * hidden < 2**24
        self.x, self.ids, self.dtype = whole(t, hidden).to(dtype), ids.int().cuda(), dtype
        self.w13, self.w2 = (torch.stack([whole(n, k).to(E4M3) for _ in range(ne)]) for n, k in ((2 * inter, hidden), (hidden, inter)))
        self.s13 = torch.full((ne, -(-2 * inter // 128), -(-hidden // 128)), 2.0**-9, device="cuda")
        self.s2 = 2e-4 * (0.5 + torch.rand(ne, -(-hidden // 128), -(-inter // 128), generator=g, device="cuda"))
        self.weights = 0.1 + torch.rand(ids.shape, generator=g, device="cuda")
        self.hidden, self.inter, self.ne = hidden, inter, ne

    def want(self):
        """The layer in float64 and the sum of magnitudes behind each result; and the operands' step bound of the second product."""
        out, size, step = (torch.zeros(self.x.shape, dtype=torch.float64, device="cuda") for _ in range(3))
        for e in range(self.ne):
            token, slot = torch.nonzero(self.ids == e, as_tuple=True)
            if len(token) == 0:
                continue
            both = self.x[token].double() @ self.w13[e].double().t() * 2.0**-9
            assert torch.equal(both.float().double(), both)
            h, hs = ops.fp8_silu_mul_quantize(both.float())
            hv = h.double() * hs.double().t().repeat_interleave(128, 1)[:, : self.inter]
            down = self.w2[e].double() * self.s2[e].double().repeat_interleave(128, 0)[: self.hidden].repeat_interleave(128, 1)[:, : self.inter]
            w = self.weights[token, slot].double()[:, None]
            out.index_add_(0, token, w * (hv @ down.t()))
            size.index_add_(0, token, w * (hv.abs() @ down.abs().t()))
            step.index_add_(0, token, w * _step_bound(hv, down))
        return out, size, step

    def check(self, y, eight_bit=False):
        out, size, step = self.want()
        # float32 sums of the second product as in _linear_bound, the weights' products and their sum, one rounding to the type
        terms = self.inter / 128 + 20 + self.ids.shape[1] + 2
        bound = size * terms * 2.0**-23 + out.abs() * UNIT[self.dtype] + 2.0**-24 * (self.dtype == torch.float16)
        err = (y.double() - out).abs()
        assert (err <= bound + (step * (1 + 2.0**-20) if eight_bit else 0)).all(), (err / bound).max()

    def run(self):
        return ops.fp8_moe_experts(self.x, self.weights, self.ids, self.w13, self.s13, self.w2, self.s2)


@pytest.mark.parametrize("hidden,inter", [(256, 8208), (4096, 14336), (512, 8320), (8208, 256), (8192, 8192), (9344, 384)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_token_beyond_the_one_row_kernel(hidden, inter, dtype):
    ne, k = 3, 2
    layer = ExactLayer(1, hidden, inter, ne, torch.tensor([[2, 0]]), dtype, top=8 if hidden < 8192 else 4)
    layer.check(layer.run())
    # the same through the C entry, in a workspace that shows what was written: no product is computed for another form to compute again
    size = _lib.lib().mi355gq_fp8_moe_workspace_bytes(1, hidden, inter, ne, k)
    space = torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(layer.x)
    _lib.call("mi355gq_fp8_moe", layer.x.data_ptr(), 1, hidden, inter, ne, k, layer.weights.data_ptr(), layer.ids.data_ptr(), layer.w13.data_ptr(),
              hidden, layer.s13.data_ptr(), layer.w2.data_ptr(), inter, layer.s2.data_ptr(), ops._MODEL_DTYPES[dtype], out.data_ptr(),
              space.data_ptr(), size, ops._stream())
    layer.check(out)
    written = int((space != 0xA5).sum())
    both = 4 * k * inter
    rest = hidden + k * inter + 4 * (hidden // 128 + 1 + k * (inter // 128 + 1) + 2 * k + ne + 1) + 4 * k * hidden
    if hidden <= 8192 and inter <= 8192:
        assert "fp8_gemv_sum" in _lib.last_kernel() and written <= both
    elif inter % 128 == 0:
        assert "fp8_rows" in _lib.last_kernel() and written <= rest, (written, rest)
    else:  # gate and up apart from the activation
        assert "fp8_rows" in _lib.last_kernel() and written <= rest + 2 * both


@pytest.mark.parametrize("rows,k,pitch", [(3, 128, 512), (5, 130, 400), (1, 1, 256), (4, 40, 48), (2, 600, 1600), (7, 136, 144)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantisers_write_their_own_bytes_alone(rows, k, pitch, dtype):
    # rows in a wider buffer, whose other bytes belong to somebody: [K, the next multiple of 8) becomes zeros, the rest stays
    x = torch.randn(rows, k, generator=_gen(k)).to(dtype).cuda()
    both = torch.randn(rows, 2 * k, generator=_gen(k)).to(dtype).cuda()
    up8 = -(-k // 8) * 8
    scale = torch.empty(-(-k // 128) * max(rows, 128), device="cuda")
    code, stream = ops._MODEL_DTYPES[dtype], ops._stream()
    calls = {"mi355gq_fp8_quantize": lambda q: (x.data_ptr(), rows, k, code, q, pitch, scale.data_ptr(), stream),
             "mi355gq_fp8_silu_mul_quantize": lambda q: (both.data_ptr(), rows, k, code, q, pitch, scale.data_ptr(), stream),
             "mi355gq_fp8_quantize_weight": lambda q: (x.data_ptr(), 1, rows, k, code, q, pitch, scale.data_ptr(), stream)}
    want = {"mi355gq_fp8_quantize": lambda: ops.fp8_quantize(x)[0], "mi355gq_fp8_silu_mul_quantize": lambda: ops.fp8_silu_mul_quantize(both)[0],
            "mi355gq_fp8_quantize_weight": lambda: ops.fp8_quantize_weight(x)[0]}
    for name, args in calls.items():
        buf = torch.full((rows + 1, pitch), 0xA5, dtype=torch.uint8, device="cuda")
        _lib.call(name, *args(buf.data_ptr()))
        assert torch.equal(buf[:rows, :k], want[name]().view(torch.uint8)[:, :k]), name
        assert (buf[:rows, k:up8] == 0).all() and (buf[:rows, up8:] == 0xA5).all() and (buf[rows] == 0xA5).all(), name


def test_layers_run_after_a_copy_and_a_move(tmp_path):
    n, k = 72, 200  # rows of 200 bytes in 208
    torch.manual_seed(0)
    src = torch.nn.Linear(k, n, dtype=torch.float16, device="cuda")
    linear = layers.Fp8Linear.from_linear(src)
    x = torch.randn(3, k, device="cuda", dtype=torch.float16)
    want = linear(x)
    on_cpu = copy.deepcopy(linear).cpu()
    fresh = layers.Fp8Linear(k, n, dtype=torch.float16)
    fresh.load_state_dict(on_cpu.state_dict())
    assigned = layers.Fp8Linear(k, n, dtype=torch.float16, device="cuda")
    assigned.load_state_dict({name: v.clone() for name, v in linear.state_dict().items()}, assign=True)
    torch.save(on_cpu, tmp_path / "layer.pt")
    loaded = torch.load(tmp_path / "layer.pt", weights_only=False)  # (written above)
    for other in (copy.deepcopy(linear), on_cpu.cuda(), fresh.cuda(), assigned, loaded.to("cuda")):
        assert torch.equal(other(x), want)


def test_layers_run_after_a_cast():
    n, k = 72, 200
    torch.manual_seed(0)
    linear = layers.Fp8Linear.from_linear(torch.nn.Linear(k, n, dtype=torch.float16, device="cuda"))
    x = torch.randn(3, k, device="cuda", dtype=torch.float16)
    assert torch.equal(copy.deepcopy(linear).half()(x), linear(x))
    both = copy.deepcopy(linear).to(torch.bfloat16)
    assert both.bias.dtype == torch.bfloat16 and both(x.bfloat16()).dtype == torch.bfloat16
    assert torch.equal(both(x.bfloat16()), ops.fp8_linear(x.bfloat16(), linear.q_weight, linear.q_scale, bias=linear.bias.bfloat16()))
    moe = layers.Fp8MoE(256, 144, 4, 2, scoring="sigmoid", score_bias=True)
    moe = moe.to("cuda", torch.float16)
    moe.load_experts(torch.randn(4, 288, 256, device="cuda") * 0.05, torch.randn(4, 256, 144, device="cuda") * 0.05)
    x, gate = torch.randn(5, 256, device="cuda", dtype=torch.float16), torch.randn(5, 4, device="cuda", dtype=torch.float16)
    want = moe(x, gate)
    assert torch.equal(copy.deepcopy(moe).half()(x, gate), want) and torch.equal(torch.nn.Sequential(moe).half()[0](x, gate), want)


def test_layer_whose_expert_spans_four_gib_by_its_pitch():
    # rows of gate and up far apart: neither fused form reaches them, product and activation go apart and need the scratch for it
    t, hidden, inter, pitch = 40, 256, 256, (1 << 23) + 16
    layer = ExactLayer(t, hidden, inter, 1, torch.zeros(t, 1), torch.float16)
    wide = torch.empty(2 * inter * pitch, dtype=torch.uint8, device="cuda").view(E4M3).as_strided((1, 2 * inter, hidden), (2 * inter * pitch, pitch, 1))
    assert 2 * inter * pitch > 2**32
    wide.copy_(layer.w13)
    want = layer.run()
    layer.w13 = wide
    got = layer.run()
    assert torch.equal(got, want)
    layer.check(got, eight_bit=True)
    # the router and the layer in one call
    logits = torch.zeros(t, 1, device="cuda")
    assert torch.equal(ops.fp8_moe(layer.x, logits, wide, layer.s13, layer.w2, layer.s2, 1),
                       ops.fp8_moe_experts(layer.x, torch.ones(t, 1, device="cuda"), layer.ids, wide, layer.s13, layer.w2, layer.s2))
    layer.x, layer.ids, layer.weights = layer.x[:1], layer.ids[:1], layer.weights[:1]  # one token
    layer.check(layer.run())


def test_linear_on_one_row_of_a_wider_matrix():
    # a single row's stride says nothing: columns of a matrix's last row, whose pitch the row's own bytes do not fill
    x = torch.randn(7, 256, generator=_gen(2)).half().cuda()
    q, s = ops.fp8_quantize(x)
    wide = torch.zeros(7, 4096, dtype=torch.uint8, device="cuda").view(E4M3)
    wide[:, 3840:] = q
    w, ws = (v.cuda() for v in _weights(64, 256, 1))
    want = ops.fp8_linear((q, s), w, ws)
    last = ops.fp8_linear((wide[6:7, 3840:], s[:, 6:7].contiguous()), w, ws)
    assert torch.equal(last, ops.fp8_linear((q[6:7].contiguous(), s[:, 6:7].contiguous()), w, ws))
    assert ((last - want[6:7]).abs() <= 2.0**-9 * want[6:7].abs() + 2.0**-10).all()
    assert torch.equal(ops.fp8_dequantize(wide[6:7, 3840:], s[:, 6:7].contiguous(), row_groups=True), ops.fp8_dequantize(q, s, row_groups=True)[6:7])


@pytest.mark.parametrize("counts,n,k,form", [([40, 0, 0, 0, 0, 0], 64, 2048, "4 blocks x 4 waves, 1 phases"), ([0, 17, 1, 0, 0, 0, 33, 0], 200, 272, None),
                                             ([0, 17, 1, 0, 0, 0, 33, 0], 130, 14336, "2 phases"), ([0] * 15 + [90], 1032, 1040, None),
                                             ([48, 0, 0, 0, 0, 0], 136, 20480, "phases"), ([16, 32, 0, 0, 0, 0, 0, 1], 36, 16, None)])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("out", DTYPES)
def test_segments_of_several_passes(counts, n, k, form, gather, out):
    rows, experts = sum(counts), len(counts)
    w, ws = _weights(n, k, 13, experts)
    indptr = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    source = max(rows // 3, 1) if gather else rows
    x = torch.randn(source, k, generator=_gen(rows + k)).to(torch.bfloat16)
    index = torch.randint(0, source, (rows,), generator=_gen(1), dtype=torch.int32) if gather else None
    q, s = ops.fp8_quantize(x.cuda())
    y = ops.fp8_group_gemm(q, s, index.cuda() if gather else None, w.cuda()[..., :k], ws.cuda(), indptr.cuda(), out).cpu().double()
    assert "fp8_rows" in _lib.last_kernel()
    if form == "phases":
        assert "1 phases" not in _lib.last_kernel()
    elif form:
        assert form in _lib.last_kernel()
    xv = quantized(x.double())[2]
    xv = xv[index.long()] if gather else xv
    for e in range(experts):
        part = slice(int(indptr[e]), int(indptr[e + 1]))
        wv = block_values(w[e, :, :k].float().nan_to_num(), ws[e])
        exact = xv[part] @ wv.t()
        assert ((y[part] - exact).abs() <= _linear_bound(xv[part], wv, exact, out)).all()


def _skewed(t, ne, k, first):
    """Expert `first` for every token, the others spread."""
    others = [e for e in range(ne) if e != first]
    return torch.tensor([[first] + [others[(i * (k - 1) + j) % len(others)] for j in range(k - 1)] for i in range(t)])


@pytest.mark.parametrize("t,hidden,inter,ne,ids,few", [
    (1, 512, 256, 8, _skewed(1, 8, 3, 5), True), (4, 512, 256, 8, _skewed(4, 8, 2, 0), True), (16, 256, 384, 64, _skewed(16, 64, 4, 63), True),
    (40, 256, 128, 64, _skewed(40, 64, 1, 7), True), (50, 384, 256, 96, _skewed(50, 96, 2, 3), True), (36, 9344, 128, 40, _skewed(36, 40, 1, 9), True),
    (40, 272, 144, 64, _skewed(40, 64, 1, 7), True), (70, 256, 128, 6, _skewed(70, 6, 2, 2), False), (300, 512, 256, 4, _skewed(300, 4, 1, 1), False),
    (130, 272, 144, 5, _skewed(130, 5, 2, 4), False)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_layer_rounds_once(t, hidden, inter, ne, ids, few, dtype):
    # skewed routing: one expert has all tokens, several passes of the few-row kernel (9344: x of a pass in two phases) or many tiles
    layer = ExactLayer(t, hidden, inter, ne, ids, dtype, top=8 if hidden < 8192 else 4)
    layer.check(layer.run(), eight_bit=not few)


@pytest.mark.parametrize("m", [2, 3, 7, 12])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [torch.inf, -torch.inf, torch.nan])
def test_few_rows_keep_what_is_not_finite_in_its_row(m, dtype, bad):
    for n, k in ((256, 512), (1000, 1040)):
        w, ws = (v.cuda() for v in _weights(n, k, 5))
        x = torch.randn(m, k, generator=_gen(6)).to(dtype)
        clean = ops.fp8_linear(x.cuda(), w, ws)
        assert "fp8_rows" in _lib.last_kernel()
        for row, at in ((0, 300), (m - 1, k - 1)):
            dirty = x.clone()
            dirty[row, at] = bad
            for y in (ops.fp8_linear(dirty.cuda(), w, ws), ops.fp8_linear(ops.fp8_quantize(dirty.cuda()), w, ws, out_dtype=dtype)):
                rest = [r for r in range(m) if r != row]
                assert y[row].isnan().all() and torch.equal(y[rest], clean[rest])


def test_more_rows_than_a_grid_holds():
    # four rows a workgroup of 256: from 2^26 rows on a launch's grid would leave 32 bits
    rows, k = (1 << 26) + 5, 16
    assert (rows + 3) // 4 * 256 > 2**32
    x = torch.randn(rows, k, device="cuda", dtype=torch.bfloat16)
    q, s = ops.fp8_quantize(x)
    back = ops.fp8_dequantize(q, s, torch.bfloat16, row_groups=True)
    for part in (slice(0, 300), slice(rows // 2 - 100, rows // 2 + 100), slice(rows - 300, rows)):
        want_q, want_s, want_v = quantized(x[part].cpu().double())
        assert torch.equal(s[0, part].cpu().double(), want_s[:, 0]) and torch.equal(q[part].cpu().double(), want_q)
        assert torch.equal(back[part].cpu(), want_v.float().bfloat16())
    # everything, by the definition of the scale: within half a step of the value, and no smaller scale would do
    for part in torch.arange(0, rows, 1 << 23).tolist():
        end = min(part + (1 << 23), rows)
        v, top, sc = x[part:end].float(), x[part:end].float().abs().amax(1), s[0, part:end]
        assert ((top <= 448 * sc) & ((top > 224 * sc) | (top == 0))).all()
        assert ((back[part:end].float() - v).abs() <= v.abs() * (2.0**-4 + 2.0**-8) + sc[:, None] * 2.0**-9).all()
    del x, back
    both = torch.randn(rows, 2 * k, device="cuda", dtype=torch.float16)
    q, s = ops.fp8_silu_mul_quantize(both)
    part = slice(rows - 300, rows)
    q2, s2 = ops.fp8_silu_mul_quantize(both[part].contiguous())
    assert torch.equal(q[part].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[:, part], s2)


def test_more_tokens_than_a_grid_holds():
    # 32 work items a token: from 2^27 tokens on a launch's grid would leave 32 bits
    t = (1 << 27) + 5
    logits = torch.randint(-3, 4, (t, 2), device="cuda", dtype=torch.int8).to(torch.bfloat16)
    weights, ids = ops.moe_gating(logits, 1, "sigmoid", renormalize=False)
    for part in torch.arange(0, t, 1 << 24).tolist():
        a, b = logits[part : part + (1 << 24)].float().unbind(1)
        assert torch.equal(ids[part : part + (1 << 24), 0], (b > a).int())  # ties keep the lower index
        assert ((weights[part : part + (1 << 24), 0] - torch.sigmoid(torch.maximum(a, b))).abs() <= 2.0**-21).all()


def test_more_tiles_than_a_grid_holds():
    # 512 experts, all but the first without rows, and so many columns that 512 tiles a column of 128 are 2^32 work items and more.  K = 8 is the
    # tiles', whatever the number of rows.  Only the first expert's weights are there: nothing reads the others'.
    rows, n, k, experts = 3, 4300000, 8, 512
    assert -(-n // 128) * experts * 256 > 2**32
    x = torch.randint(-8, 9, (rows, k), device="cuda").half()
    q, s = ops.fp8_quantize(x)
    w = torch.zeros(n, 16, dtype=torch.uint8, device="cuda").view(E4M3)
    w[:, :k] = torch.randint(-8, 9, (n, k), device="cuda", dtype=torch.int8).half().to(E4M3)
    ws = torch.full((-(-n // 128), 1), 0.5, device="cuda")
    indptr = torch.full((experts + 1,), rows, dtype=torch.int32, device="cuda")
    indptr[0] = 0
    want = (x.float() @ w[:, :k].float().t().contiguous()) * 0.5  # whole numbers: exact in any order
    for precise in (0, 1):
        y = torch.full((rows, n), -1e9, device="cuda")
        _lib.call("mi355gq_fp8_group_gemm", q.data_ptr(), 16, s.data_ptr(), rows, None, rows, w.data_ptr(), 16, ws.data_ptr(), indptr.data_ptr(), experts,
                  n, k, ops._MODEL_DTYPES[torch.float32], precise, y.data_ptr(), ops._stream())
        assert "fp8_tile" in _lib.last_kernel() and torch.equal(y, want)


@pytest.mark.parametrize("spread,documented", [(0.0, 1.5e-5), (0.7, 2.7e-5), (2.0, 7.7e-5)])
@pytest.mark.parametrize("m,n,k", [(24, 1024, 4096), (300, 1024, 14336), (512, 1024, 768)])
def test_what_the_8_bit_instruction_drops(m, n, k, spread, documented):
    # the documented error of a whole result, normal weights and x's channels spread by exp(spread N), which other seeds move little
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp(spread * torch.randn(k, generator=g, device="cuda"))
    w = (100 * torch.randn(n, k, generator=g, device="cuda")).clamp(-448, 448).to(E4M3)
    ws = 2e-4 * (0.5 + torch.rand(-(-n // 128), k // 128, generator=g, device="cuda"))
    q, s = ops.fp8_quantize(x)
    wv = w.double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)
    exact = torch.matmul(q.double() * s.double().t().repeat_interleave(128, 1), wv.t().contiguous())
    for precise, most in ((False, 2 * documented), (True, 4e-7)):
        y = ops.fp8_linear((q, s), w, ws, out_dtype=torch.float32, precise=precise).double()
        assert (y - exact).norm() <= most * exact.norm()


@pytest.mark.parametrize("t", [1, 5, 40])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_layer_on_x_at_an_odd_offset(t, dtype):
    layer = ExactLayer(t, 256, 128, 8, _skewed(t, 8, 2, 3), dtype)
    want = layer.run()
    flat = torch.empty(layer.x.numel() + 1, dtype=dtype, device="cuda")
    flat[1:] = layer.x.flatten()
    odd = flat[1:].view(t, 256)
    assert odd.data_ptr() % 16 and odd.is_contiguous()
    logits = torch.randn(t, 8, generator=_gen(t)).cuda()
    args = (logits, layer.w13, layer.s13, layer.w2, layer.s2, 2)
    assert torch.equal(ops.fp8_moe(odd, *args), ops.fp8_moe(layer.x, *args))
    layer.x = odd
    assert torch.equal(layer.run(), want)


@pytest.mark.parametrize("t", [1, 5, 40])
def test_layer_in_place(t):
    layer = ExactLayer(t, 256, 128, 8, _skewed(t, 8, 2, 3), torch.float16)
    want, x = layer.run(), layer.x.clone()
    size = _lib.lib().mi355gq_fp8_moe_workspace_bytes(t, 256, 128, 8, 2)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    _lib.call("mi355gq_fp8_moe", x.data_ptr(), t, 256, 128, 8, 2, layer.weights.data_ptr(), layer.ids.data_ptr(), layer.w13.data_ptr(), 256,
              layer.s13.data_ptr(), layer.w2.data_ptr(), 128, layer.s2.data_ptr(), ops._MODEL_DTYPES[torch.float16], x.data_ptr(), space.data_ptr(), size,
              ops._stream())
    assert torch.equal(x, want)
