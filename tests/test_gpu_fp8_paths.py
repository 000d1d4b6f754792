"""Every path of the 8-bit block-scaled operators: the tile forms and their shares of K, waves without rows, a product whose last round is a
form of its own, routing over every split of experts into groups, the native call path, and the layers that run them together."""

import pytest
import torch

from mlc_llm_amd import _lib, nn as layers, ops
from test_gpu_fp8 import _gen, _linear_bound, _step_bound, _weights, block_values, quantized, route
from test_native_call import Plain

pytestmark = pytest.mark.gpu


@pytest.fixture
def options():
    def choose(form=-1, shares=-1):
        _lib.set_option("gemm_variant", form)
        _lib.set_option("gemm_split_k", shares)

    yield choose
    choose()


def _check(y, xv, wv, bias=None):
    exact = xv @ wv.t()
    bound = _linear_bound(xv, wv, exact, torch.bfloat16) + _step_bound(xv, wv)
    if bias is not None:
        exact = exact + bias.double()
        bound = bound + (exact.abs() + bias.double().abs()) * (2.0**-8 + 2.0**-22)
    err = (y.double() - exact).abs()
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("form", range(6))
@pytest.mark.parametrize("m,n,k", [(18, 136, 528), (70, 260, 1040), (200, 392, 1536), (300, 520, 2064)])
def test_tile_forms_and_shares(options, form, m, n, k):
    g = _gen(m + n)
    x = torch.randn(m, k, generator=g).to(torch.bfloat16).cuda()
    w, ws = _weights(n, k, 3)
    bias = torch.randn(n, generator=g).to(torch.bfloat16).cuda()
    wd, wsd = w.cuda()[:, :k], ws.cuda()
    xv, wv = quantized(x.cpu().double())[2].cuda(), block_values(w[:, :k].float().nan_to_num(), ws).cuda()
    for shares in (1, 2, 3, 4):
        if shares > 1 and -(-k // 128) < 4 * shares:
            continue
        options(form, shares)
        y = ops.fp8_linear(x, wd, wsd, bias=bias)
        assert "%d shares" % shares in _lib.last_kernel()
        _check(y, xv, wv, bias)
        assert torch.equal(y, ops.fp8_linear(x, wd, wsd, bias=bias))


@pytest.mark.parametrize("form", range(3))
@pytest.mark.parametrize("m,n,k", [(18, 136, 528), (70, 260, 1040), (200, 392, 1536), (300, 520, 2064)])
def test_precise_forms_and_shares(options, form, m, n, k):
    x = torch.randn(m, k, generator=_gen(m + n))
    w, ws = _weights(n, k, 3)
    residual = torch.randn(m, n, generator=_gen(m))
    wd, wsd = w.cuda()[:, :k], ws.cuda()
    xv, wv = quantized(x.double())[2].cuda(), block_values(w[:, :k].float().nan_to_num(), ws).cuda()
    exact = xv @ wv.t() + residual.cuda().double()
    for shares in (1, 2, 3, 4):
        if shares > 1 and -(-k // 128) < 4 * shares:
            continue
        options(form, shares)
        y = ops.fp8_linear(x.cuda(), wd, wsd, residual=residual.cuda())
        assert "float32 sums, %d shares" % shares in _lib.last_kernel()
        bound = _linear_bound(xv, wv, exact, torch.float32) + (exact.abs() + residual.cuda().double().abs()) * 2.0**-22
        assert ((y.double() - exact).abs() <= bound).all()


def test_last_round_in_a_form_of_its_own(options):
    m, n, k = 1024, 16500, 1024
    x = torch.randn(m, k, generator=_gen(1)).to(torch.bfloat16).cuda()
    w, ws = (t.cuda() for t in _weights(n, k, 2))
    residual = torch.randn(m, n, generator=_gen(4)).to(torch.bfloat16).cuda()
    y = ops.fp8_linear(x, w, ws, residual=residual)
    assert "256x256" not in _lib.last_kernel()  # the second launch
    options(0, 1)
    whole = ops.fp8_linear(x, w, ws, residual=residual)
    assert "256x256" in _lib.last_kernel()
    # a form takes a block's sum in one instruction and blocks in their order, whatever its size
    assert torch.equal(y, whole)
    xv = quantized(x.cpu().double())[2].cuda()
    for part in (slice(0, 128), slice(16256, n)):  # a column of tiles ends at 16384
        wv = block_values(w.cpu().float()[part], ws.cpu()[part.start // 128 : -(-part.stop // 128)]).cuda()
        exact = xv @ wv.t() + residual[:, part].double()
        bound = _linear_bound(xv, wv, exact, torch.bfloat16) + _step_bound(xv, wv) + (exact.abs() + residual[:, part].double().abs()) * 2.0**-22
        assert ((y[:, part].double() - exact).abs() <= bound).all()


@pytest.mark.parametrize("form", range(6))
@pytest.mark.parametrize("counts", [[33, 1, 0, 64, 65, 257], [20] * 7, [16, 48, 130, 191]])
def test_segments_that_leave_waves_without_rows(options, form, counts):
    n, k, experts, rows = 264, 400, len(counts), sum(counts)
    w, ws = _weights(n, k, 11, experts)
    indptr = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    x = torch.randn(40, k, generator=_gen(rows)).to(torch.bfloat16)
    index = torch.randint(0, 40, (rows,), generator=_gen(1), dtype=torch.int32)
    q, s = ops.fp8_quantize(x.cuda())
    options(form)
    y = ops.fp8_group_gemm(q, s, index.cuda(), w.cuda()[..., :k], ws.cuda(), indptr.cuda(), torch.bfloat16).cpu()
    assert "fp8_tile" in _lib.last_kernel()
    xv = quantized(x.double())[2][index.long()]
    for e in range(experts):
        part = slice(int(indptr[e]), int(indptr[e + 1]))
        _check(y[part], xv[part], block_values(w[e, :, :k].float().nan_to_num(), ws[e]))


@pytest.mark.parametrize("k", [16, 112, 1024, 4112, 8192, 8208, 14336])
@pytest.mark.parametrize("n", [1, 130, 1032])
def test_one_row(n, k):
    x = torch.randn(1, k, generator=_gen(k)).to(torch.float16)
    w, ws = _weights(n, k, 5)
    xv, wv = quantized(x.double())[2], block_values(w[:, :k].float().nan_to_num(), ws)
    exact = xv @ wv.t()
    wd, wsd = w.cuda()[:, :k], ws.cuda()
    y = ops.fp8_linear(x.cuda(), wd, wsd, out_dtype=torch.float32)
    assert ((y.cpu().double() - exact).abs() <= _linear_bound(xv, wv, exact, torch.float32)).all()
    y = ops.fp8_linear(ops.fp8_quantize(x.cuda()), wd, wsd, out_dtype=torch.float32, precise=True)
    assert ((y.cpu().double() - exact).abs() <= _linear_bound(xv, wv, exact, torch.float32)).all()


@pytest.mark.parametrize("ne,groups,top_groups", [(16, 16, 5), (48, 16, 3), (96, 32, 9), (128, 64, 8), (160, 8, 3), (160, 5, 2), (256, 8, 4), (256, 2, 1), (260, 4, 2),
                                                  (320, 64, 40), (512, 4, 3), (512, 1, 1), (72, 1, 1)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gating_over_groups(ne, groups, top_groups, bias, dtype):
    k = min(8, ne // groups * top_groups)
    logits = torch.randn(37, ne, generator=_gen(ne + groups)).to(dtype)
    b = 0.1 * torch.randn(ne, generator=_gen(7)) if bias else None
    weights, ids = ops.moe_gating(logits.cuda(), k, "sigmoid", b.cuda() if bias else None, groups, top_groups, True, 2.5)
    want_w, want_ids = route(logits, b, k, "sigmoid", groups, top_groups, True, 2.5)
    # a choice that hangs on the last bits of a key may go either way: such tokens are left out, and are few
    same = (ids.cpu().long() == want_ids).all(1)
    assert same.float().mean() >= 0.9
    assert ((weights.cpu().double() - want_w)[same].abs() <= 2.0**-20 * want_w[same]).all()


def test_a_row_of_unaligned_logits():
    logits = torch.randn(9 * 64 + 1, generator=_gen(3)).to(torch.bfloat16).cuda()
    odd = logits[1:].view(9, 64)
    w, ids = ops.moe_gating(odd, 6)
    w2, ids2 = ops.moe_gating(odd.clone(), 6)
    assert torch.equal(w, w2) and torch.equal(ids, ids2)
    odd = logits[1 : 1 + 4 * 128].view(4, 128)
    w, ids = ops.moe_gating(odd, 32)
    w2, ids2 = ops.moe_gating(odd.clone(), 32)
    assert torch.equal(w, w2) and torch.equal(ids, ids2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t", [0, 1, 5, 40])
def test_native_and_python_routes_agree(dtype, t):
    native = _lib.native()
    x = torch.randn(t, 384, generator=_gen(t)).to(dtype).cuda()
    w, ws = (v.cuda() for v in _weights(200, 384, 1))
    plain = x.as_subclass(Plain)
    assert t == 0 or native.fp8_quantize(x) is not None
    for a, b in zip(ops.fp8_quantize(x), ops.fp8_quantize(plain)):
        assert a.shape == b.shape and (t == 0 or torch.equal(a.view(torch.uint8), b.as_subclass(torch.Tensor).view(torch.uint8))) and a.stride() == b.stride()
    bias, residual = torch.randn(200).to(dtype).cuda(), torch.randn(t, 200).to(dtype).cuda()
    for out in (None, torch.float32):
        for b, r in ((None, None), (bias, None), (None, residual), (bias, residual)):
            assert t == 0 or native.fp8_linear(x, w, ws, b, out, r, None) is not None
            got, want = ops.fp8_linear(x, w, ws, b, out, r), ops.fp8_linear(plain, w, ws, b, out, r)
            assert got.dtype == want.dtype and torch.equal(got, want.as_subclass(torch.Tensor))
    logits = torch.randn(t, 16, generator=_gen(9)).cuda()
    for a, b in zip(ops.moe_gating(logits, 3), ops.moe_gating(logits.as_subclass(Plain), 3)):
        assert torch.equal(a, b.as_subclass(torch.Tensor))
    w13, s13 = (v.cuda() for v in _weights(512, 384, 2, 16))
    w2, s2 = (v.cuda() for v in _weights(384, 256, 3, 16))
    got, want = ops.fp8_moe(x, logits, w13, s13, w2, s2, 3), ops.fp8_moe(plain, logits, w13, s13, w2, s2, 3)
    assert got.shape == x.shape and torch.equal(got, want.as_subclass(torch.Tensor))


def test_layers_run_the_operators():
    torch.manual_seed(0)
    src = torch.nn.Linear(400, 264, dtype=torch.bfloat16, device="cuda")
    linear = layers.Fp8Linear.from_linear(src)
    x = torch.randn(2, 5, 400, device="cuda", dtype=torch.bfloat16)
    want = ops.fp8_linear(x, *ops.fp8_quantize_weight(src.weight.detach()), bias=src.bias.detach())
    assert torch.equal(linear(x), want)
    again = layers.Fp8Linear(400, 264, dtype=torch.bfloat16, device="cuda")
    again.load_state_dict(linear.state_dict())
    assert again.q_weight.stride() == (400, 1) and torch.equal(again(x, residual=want), linear(x, residual=want))
    moe = layers.Fp8MoE(256, 144, 16, 4, scoring="sigmoid", score_bias=True, num_groups=4, top_groups=2, routed_scale=2.5, device="cuda")
    e1_e3, e2 = torch.randn(16, 288, 256, device="cuda") * 0.05, torch.randn(16, 256, 144, device="cuda") * 0.05
    moe.load_experts(e1_e3, e2)
    moe.score_bias.data.copy_(0.1 * torch.randn(16))
    w13, s13 = ops.fp8_quantize_weight(e1_e3)
    w2, s2 = ops.fp8_quantize_weight(e2)
    for lead in ((1, 1), (3, 7), (1, 130)):
        x = torch.randn(*lead, 256, device="cuda", dtype=torch.float16)
        gate = torch.randn(lead[0] * lead[1], 16, device="cuda", dtype=torch.float16)
        y = moe(x, gate)
        weights, ids = ops.moe_gating(gate, 4, "sigmoid", moe.score_bias, 4, 2, True, 2.5)
        assert y.shape == x.shape and torch.equal(y.view(-1, 256), ops.fp8_moe_experts(x.view(-1, 256), weights, ids, w13, s13, w2, s2))


@pytest.mark.parametrize("t,ne,k", [(1100, 3, 2), (600, 2, 1), (300, 2, 2), (770, 3, 3)])
def test_layers_of_many_rows_an_expert(t, ne, k):
    # the gate/up product in both of its forms, tiles that end in every row of waves, against the two steps on their own
    hidden, inter = 400, 256
    x = torch.randn(t, hidden, generator=_gen(t)).to(torch.float16).cuda()
    logits = torch.randn(t, ne, generator=_gen(t + 1)).cuda()
    w13, s13 = (v.cuda() for v in _weights(2 * inter, hidden, 2, ne))
    w2, s2 = (v.cuda() for v in _weights(hidden, inter, 3, ne))
    weights, ids = ops.moe_gating(logits, k)
    row_token, slot_row, indptr = ops.moe_plan(ids, ne)
    q, s = ops.fp8_quantize(x)
    both = ops.fp8_group_gemm(q, s, row_token, w13, s13, indptr, torch.float32, True)
    h, hs = ops.fp8_silu_mul_quantize(both)
    y = ops.fp8_group_gemm(h, hs, None, w2, s2, indptr, torch.float32, False).double()
    want = (y[slot_row.view(t, k).long()] * weights.double()[..., None]).sum(1)
    got = ops.fp8_moe_experts(x, weights, ids, w13, s13, w2, s2)
    size = (y[slot_row.view(t, k).long()].abs() * weights.double()[..., None]).sum(1)
    assert ((got.double() - want).abs() <= 2.0**-11 * want.abs() + size * (k + 2) * 2.0**-23 + 2.0**-24).all()


def test_weights_beyond_four_gib():
    n, k = 262144 + 4096, 16384
    w = torch.randint(0, 0x78, (n, k), dtype=torch.uint8, device="cuda")  # no NaN
    w[:, ::3] |= 0x80
    w = w.view(torch.float8_e4m3fn)
    ws = 2e-4 * (0.5 + torch.rand(-(-n // 128), k // 128, device="cuda"))
    assert w.numel() > 2**32
    for m in (1, 8, 20):
        x = torch.randn(m, k, generator=_gen(m)).to(torch.bfloat16).cuda()
        y = ops.fp8_linear(x, w, ws, out_dtype=torch.float32)
        xv = quantized(x.cpu().double())[2].cuda()
        for part in (slice(0, 256), slice(131072, 131072 + 256), slice(n - 256, n)):
            wv = block_values(w[part].float(), ws[part.start // 128 : part.stop // 128])
            exact = xv @ wv.t()
            assert ((y[:, part].double() - exact).abs() <= _linear_bound(xv, wv, exact, torch.float32)).all()
    # the same bytes as a stack of experts, a few rows and many rows each
    experts = 65
    stack, scales = w.view(experts, n // experts, k), ws.view(experts, n // experts // 128, k // 128)
    for each in (3, 40):
        indptr = torch.arange(experts + 1, dtype=torch.int32).cuda() * each
        x = torch.randn(experts * each, k, generator=_gen(each)).to(torch.bfloat16).cuda()
        y = ops.fp8_group_gemm(*ops.fp8_quantize(x), None, stack, scales, indptr, torch.float32)
        for e in (0, 64):
            xv = quantized(x[e * each : e * each + each].cpu().double())[2].cuda()
            wv = block_values(stack[e, :256].float(), scales[e, :2])
            exact = xv @ wv.t()
            assert ((y[e * each : e * each + each, :256].double() - exact).abs() <= _linear_bound(xv, wv, exact, torch.float32)).all()
