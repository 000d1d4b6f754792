"""Destination-passing operators over torch ROCm tensors.

Each function plays the role the Relax VM plays around `call_dps_packed`: it
checks shapes and dtypes, allocates the output tensor(s) and hands raw pointers
plus the current HIP stream to the C ABI.  uint32 storage is held in int32
torch tensors (same bits; torch's uint32 support on device is partial).

linear, linear_silu_mul and embedding_take first offer their arguments to the native call path (csrc/gq_torch.cc), which does the
same checks, allocation and call in one step; it declines (None) whatever it does not recognise, and the Python below decides.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib


def _stream() -> int:
    native = _lib.native()
    return native.stream() if native is not None else torch.cuda.current_stream().cuda_stream


def _chk(t: torch.Tensor, dtype, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name}: must live on the GPU (got {t.device})")
    dtypes = dtype if isinstance(dtype, tuple) else (dtype,)
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype}, expected {dtypes}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    return t


_STORAGE = (torch.int32, torch.uint32)
# model dtypes of the reference's group-quant registry -> the C ABI's dtype codes
_MODEL_DTYPES = {torch.float16: _lib.F16, torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}
_FLOATS = tuple(_MODEL_DTYPES)


def num_group(k: int, group_size: int) -> int:
    return -(-k // group_size)


def num_storage(k: int, bits: int, group_size: int) -> int:
    return (group_size // (32 // bits)) * num_group(k, group_size)


def quantize(w: torch.Tensor, bits: int, group_size: int, round_mode: int = _lib.ROUND_HALF_AWAY
             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """w [..., K] in the model dtype (float16, or float32 / bfloat16 for the q4f32 / q4bf16 schemes)
    -> (q_weight int32-as-uint32 [..., nw], q_scale [..., ng] in the same dtype)."""
    _chk(w, _FLOATS, "w")
    k = w.shape[-1]
    rows = w.numel() // k if k else 0
    lead = tuple(w.shape[:-1])
    qw = torch.empty((*lead, num_storage(k, bits, group_size)), dtype=torch.int32, device=w.device)
    qs = torch.empty((*lead, num_group(k, group_size)), dtype=w.dtype, device=w.device)
    if w.dtype == torch.float16:
        _lib.call("mi355gq_quantize", w.data_ptr(), rows, k, bits, group_size, round_mode,
                  qw.data_ptr(), qs.data_ptr(), _stream())
    else:
        _lib.call("mi355gq_quantize_dt", w.data_ptr(), rows, k, bits, group_size, round_mode,
                  _MODEL_DTYPES[w.dtype], qw.data_ptr(), qs.data_ptr(), _stream())
    return qw, qs


def dequantize(q_weight: torch.Tensor, q_scale: torch.Tensor, k: int, bits: int, group_size: int
               ) -> torch.Tensor:
    """(q_weight, q_scale) -> [..., K] in the dtype of q_scale (the scheme's model dtype)."""
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, _FLOATS, "q_scale")
    lead = tuple(q_weight.shape[:-1])
    _check_qshapes(q_weight, q_scale, lead, k, bits, group_size)
    rows = 1
    for d in lead:
        rows *= d
    out = torch.empty((*lead, k), dtype=q_scale.dtype, device=q_weight.device)
    if q_scale.dtype == torch.float16:
        _lib.call("mi355gq_dequantize", q_weight.data_ptr(), q_scale.data_ptr(), rows, k, bits,
                  group_size, out.data_ptr(), _stream())
    else:
        _lib.call("mi355gq_dequantize_dt", q_weight.data_ptr(), q_scale.data_ptr(), rows, k, bits,
                  group_size, _MODEL_DTYPES[q_scale.dtype], out.data_ptr(), _stream())
    return out


def _check_qshapes(q_weight, q_scale, lead, k, bits, group_size):
    nw, ng = num_storage(k, bits, group_size), num_group(k, group_size)
    if tuple(q_weight.shape) != (*lead, nw):
        raise ValueError(f"q_weight shape {tuple(q_weight.shape)}, expected {(*lead, nw)}")
    if tuple(q_scale.shape) != (*lead, ng):
        raise ValueError(f"q_scale shape {tuple(q_scale.shape)}, expected {(*lead, ng)}")


def embedding_take(ids: torch.Tensor, q_weight: torch.Tensor, q_scale: torch.Tensor, k: int,
                   bits: int, group_size: int) -> torch.Tensor:
    native = _lib.native()
    done = native.embedding_take(ids, q_weight, q_scale, k, bits, group_size) if native is not None else None
    if isinstance(done, torch.Tensor):
        return done
    if done is not None:
        raise _lib.failed("mi355gq_embedding_take_dt", done)
    _chk(ids, torch.int32, "ids")
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, _FLOATS, "q_scale")
    num = q_weight.shape[0]
    _check_qshapes(q_weight, q_scale, (num,), k, bits, group_size)
    t = ids.numel()
    out = torch.empty((*ids.shape, k), dtype=q_scale.dtype, device=q_weight.device)
    if q_scale.dtype == torch.float16:
        _lib.call("mi355gq_embedding_take", ids.data_ptr(), t, q_weight.data_ptr(), q_scale.data_ptr(),
                  num, k, bits, group_size, out.data_ptr(), _stream())
    else:
        _lib.call("mi355gq_embedding_take_dt", ids.data_ptr(), t, q_weight.data_ptr(), q_scale.data_ptr(),
                  num, k, bits, group_size, _MODEL_DTYPES[q_scale.dtype], out.data_ptr(), _stream())
    return out


def linear(x: torch.Tensor, q_weight: torch.Tensor, q_scale: torch.Tensor, bits: int,
           group_size: int, bias: Optional[torch.Tensor] = None, out_dtype=torch.float16,
           out: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[..., N] = x[..., K] . dequantize(q_weight, q_scale)^T (+ bias) (+ residual[..., N]).

    `residual` (fp16, the shape of y) is added inside the kernel; passing the same tensor as `out`
    updates it in place."""
    native = _lib.native()
    done = native.linear(x, q_weight, q_scale, bits, group_size, bias, out_dtype, out, residual) if native is not None else None
    if isinstance(done, torch.Tensor):
        return done
    if done is not None:
        raise _lib.failed("mi355gq_linear_dt" if residual is None else "mi355gq_linear_residual_dt", done)
    _chk(x, _FLOATS, "x")
    if x.dtype != torch.float16:
        return _linear_other_dtype(x, q_weight, q_scale, bits, group_size, bias, out_dtype, out, residual)
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, torch.float16, "q_scale")
    k = x.shape[-1]
    n = q_weight.shape[0]
    _check_qshapes(q_weight, q_scale, (n,), k, bits, group_size)
    m = 1
    for d in x.shape[:-1]:
        m *= d
    if bias is not None:
        _chk(bias, torch.float16, "bias")
        if tuple(bias.shape) != (n,):
            raise ValueError(f"bias shape {tuple(bias.shape)}, expected {(n,)}")
    if out_dtype not in (torch.float16, torch.float32):
        raise TypeError(f"out_dtype {out_dtype}")
    if out is None:
        out = torch.empty((*x.shape[:-1], n), dtype=out_dtype, device=x.device)
    else:
        _chk(out, out_dtype, "out")
    if residual is not None:
        _chk(residual, torch.float16, "residual")
        if tuple(residual.shape) != tuple(out.shape) or not residual.is_contiguous():
            raise ValueError(f"residual shape {tuple(residual.shape)}, expected contiguous {tuple(out.shape)}")
    ws_bytes = _lib.lib().mi355gq_linear_workspace_bytes(m, n, k, bits, group_size)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    tail = (m, n, k, bits, group_size, _lib.F32 if out_dtype == torch.float32 else _lib.F16, out.data_ptr(),
            ws.data_ptr() if ws is not None else None, ws_bytes, _stream())
    head = (x.data_ptr(), q_weight.data_ptr(), q_scale.data_ptr(), bias.data_ptr() if bias is not None else None)
    if residual is None:
        _lib.call("mi355gq_linear", *head, *tail)
    else:
        _lib.call("mi355gq_linear_residual", *head, residual.data_ptr(), *tail)
    return out


def _check_kn_shapes(q_weight, q_scale, k, bits, group_size):
    ng = -(-k // group_size)
    nw = (group_size // (32 // bits)) * ng
    if q_weight.dim() != 2 or q_scale.dim() != 2 or q_weight.shape[0] != nw or q_scale.shape[0] != ng or \
            q_weight.shape[1] != q_scale.shape[1]:
        raise ValueError(f"KN layout: q_weight {tuple(q_weight.shape)} / q_scale {tuple(q_scale.shape)}, expected "
                         f"({nw}, N) / ({ng}, N) for K={k}")
    if not (q_weight.is_contiguous() and q_scale.is_contiguous()):
        raise ValueError("KN layout: q_weight and q_scale must be contiguous")
    return q_weight.shape[1]


def linear_kn(x: torch.Tensor, q_weight: torch.Tensor, q_scale: torch.Tensor, bits: int, group_size: int,
              bias: Optional[torch.Tensor] = None, out_dtype=torch.float16) -> torch.Tensor:
    """linear() on KN-layout tensors as a q4f16_0 / q3f16_0 model stores them: q_weight [nw, N], q_scale [ng, N]
    (float16 models).  Up to 8 rows stream them in place; more rows run on an NK copy made in a workspace."""
    _chk(x, torch.float16, "x")
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, torch.float16, "q_scale")
    k = x.shape[-1]
    n = _check_kn_shapes(q_weight, q_scale, k, bits, group_size)
    m = 1
    for d in x.shape[:-1]:
        m *= d
    if bias is not None:
        _chk(bias, torch.float16, "bias")
        if tuple(bias.shape) != (n,):
            raise ValueError(f"bias shape {tuple(bias.shape)}, expected {(n,)}")
    if out_dtype not in (torch.float16, torch.float32):
        raise TypeError(f"out_dtype {out_dtype}")
    out = torch.empty((*x.shape[:-1], n), dtype=out_dtype, device=x.device)
    ws_bytes = _lib.lib().mi355gq_linear_kn_workspace_bytes(m, n, k, bits, group_size)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    _lib.call("mi355gq_linear_kn", x.data_ptr(), q_weight.data_ptr(), q_scale.data_ptr(),
              bias.data_ptr() if bias is not None else None, m, n, k, bits, group_size,
              _lib.F32 if out_dtype == torch.float32 else _lib.F16, out.data_ptr(),
              ws.data_ptr() if ws is not None else None, ws_bytes, _stream())
    return out


def kn_to_nk(q_weight: torch.Tensor, q_scale: torch.Tensor, k: int, bits: int, group_size: int):
    """KN-layout tensors (q_weight [nw, N], q_scale [ng, N]) -> the NK tensors every other entry point takes."""
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, torch.float16, "q_scale")
    n = _check_kn_shapes(q_weight, q_scale, k, bits, group_size)
    qw = torch.empty((n, q_weight.shape[0]), dtype=torch.int32, device=q_weight.device)
    qs = torch.empty((n, q_scale.shape[0]), dtype=torch.float16, device=q_weight.device)
    _lib.call("mi355gq_kn_to_nk", q_weight.data_ptr(), q_scale.data_ptr(), n, k, bits, group_size, qw.data_ptr(),
              qs.data_ptr(), _stream())
    return qw, qs


def nk_to_kn(q_weight: torch.Tensor, q_scale: torch.Tensor, k: int, bits: int, group_size: int):
    """NK tensors (q_weight [N, nw], q_scale [N, ng]) -> the KN layout of the `_0` schemes."""
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, torch.float16, "q_scale")
    n = q_weight.shape[0]
    _check_qshapes(q_weight, q_scale, (n,), k, bits, group_size)
    qw = torch.empty((q_weight.shape[1], n), dtype=torch.int32, device=q_weight.device)
    qs = torch.empty((q_scale.shape[1], n), dtype=torch.float16, device=q_weight.device)
    _lib.call("mi355gq_nk_to_kn", q_weight.data_ptr(), q_scale.data_ptr(), n, k, bits, group_size, qw.data_ptr(),
              qs.data_ptr(), _stream())
    return qw, qs


def dequantize_kn(q_weight: torch.Tensor, q_scale: torch.Tensor, k: int, bits: int, group_size: int) -> torch.Tensor:
    """GroupQuantize._dequantize along axis 0: KN tensors -> float16 [K, N]."""
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, torch.float16, "q_scale")
    n = _check_kn_shapes(q_weight, q_scale, k, bits, group_size)
    out = torch.empty((k, n), dtype=torch.float16, device=q_weight.device)
    _lib.call("mi355gq_dequantize_kn", q_weight.data_ptr(), q_scale.data_ptr(), n, k, bits, group_size, out.data_ptr(),
              _stream())
    return out


def _linear_other_dtype(x, q_weight, q_scale, bits, group_size, bias, out_dtype, out, residual):
    """linear() for float32 / bfloat16 models: x, q_scale and bias share the model dtype; the output is
    that dtype (the default here, whatever `out_dtype` defaults to for float16) or float32."""
    dt = x.dtype
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, dt, "q_scale")
    k = x.shape[-1]
    n = q_weight.shape[0]
    _check_qshapes(q_weight, q_scale, (n,), k, bits, group_size)
    m = 1
    for d in x.shape[:-1]:
        m *= d
    if bias is not None:
        _chk(bias, dt, "bias")
        if tuple(bias.shape) != (n,):
            raise ValueError(f"bias shape {tuple(bias.shape)}, expected {(n,)}")
    if out_dtype == torch.float16:  # the float16 default of the signature
        out_dtype = dt
    if out_dtype not in (dt, torch.float32):
        raise TypeError(f"out_dtype {out_dtype} for a {dt} model")
    if out is None:
        out = torch.empty((*x.shape[:-1], n), dtype=out_dtype, device=x.device)
    else:
        _chk(out, out_dtype, "out")
    if residual is not None:
        _chk(residual, dt, "residual")
        if tuple(residual.shape) != tuple(out.shape) or not residual.is_contiguous():
            raise ValueError(f"residual shape {tuple(residual.shape)}, expected contiguous {tuple(out.shape)}")
    ws_bytes = _lib.lib().mi355gq_linear_dt_workspace_bytes(m, n, k, bits, group_size, _MODEL_DTYPES[dt])
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    head = (x.data_ptr(), q_weight.data_ptr(), q_scale.data_ptr(), bias.data_ptr() if bias is not None else None)
    tail = (m, n, k, bits, group_size, _MODEL_DTYPES[dt], _MODEL_DTYPES[out_dtype], out.data_ptr(),
            ws.data_ptr() if ws is not None else None, ws_bytes, _stream())
    if residual is None:
        _lib.call("mi355gq_linear_dt", *head, *tail)
    else:
        _lib.call("mi355gq_linear_residual_dt", *head, residual.data_ptr(), *tail)
    return out


def _unsupported(err: _lib.Mi355gqError) -> bool:
    return err.code == _lib.ERR_UNSUPPORTED


def linear_silu_mul(x: torch.Tensor, q_weight: torch.Tensor, q_scale: torch.Tensor, bits: int,
                    group_size: int) -> torch.Tensor:
    """silu(x1) * x2 with x1, x2 = split(linear(x), 2, axis=-1): the gate_up projection of an MLP
    with its activation folded into the matmul kernel.  Bit-identical to linear then silu_mul;
    shapes without a fused kernel run exactly those two calls."""
    native = _lib.native()
    done = native.linear_silu_mul(x, q_weight, q_scale, bits, group_size) if native is not None else None
    if isinstance(done, torch.Tensor):
        return done
    if done is not None and done != _lib.ERR_UNSUPPORTED:
        raise _lib.failed("mi355gq_linear_silu_mul_dt", done)
    _chk(x, _FLOATS, "x")
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, x.dtype, "q_scale")
    k = x.shape[-1]
    n = q_weight.shape[0]
    _check_qshapes(q_weight, q_scale, (n,), k, bits, group_size)
    if n % 2:
        raise ValueError(f"linear_silu_mul: {n} rows cannot be split into gate and up halves")
    m = 1
    for d in x.shape[:-1]:
        m *= d
    out = torch.empty((*x.shape[:-1], n // 2), dtype=x.dtype, device=x.device)
    dt = _MODEL_DTYPES[x.dtype]
    ws_bytes = _lib.lib().mi355gq_linear_silu_mul_dt_workspace_bytes(m, n, k, bits, group_size, dt)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    try:
        _lib.call("mi355gq_linear_silu_mul_dt", x.data_ptr(), q_weight.data_ptr(), q_scale.data_ptr(), m, n, k,
                  bits, group_size, dt, out.data_ptr(), ws.data_ptr() if ws is not None else None, ws_bytes,
                  _stream())
    except _lib.Mi355gqError as err:
        if not _unsupported(err):
            raise
        return silu_mul(linear(x.reshape(m, k), q_weight, q_scale, bits, group_size)).reshape(out.shape)
    return out


def moe_gemv_routed_silu_mul(x: torch.Tensor, gate_logits: torch.Tensor, top_k: int, q_weight: torch.Tensor,
                             q_scale: torch.Tensor, bits: int, group_size: int):
    """One token: gating_softmax_topk and the e1_e3 expert matmul with silu(x1) * x3 folded in, in one launch.
    x [1, K], gate_logits [1, num_experts] (model dtype), q_weight [E, N, nw], q_scale [E, N, ng].  Returns
    (out [top_k, N / 2], expert_weights [1, top_k], expert_ids int32 [1, top_k]); raises Mi355gqError with
    ERR_UNSUPPORTED where the fused kernel does not apply (float32 models, top_k > 2, more than 64 experts)."""
    _chk(x, _FLOATS, "x")
    _chk(gate_logits, x.dtype, "gate_logits")
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, x.dtype, "q_scale")
    if x.dim() != 2 or x.shape[0] != 1 or gate_logits.dim() != 2 or gate_logits.shape[0] != 1:
        raise ValueError("moe_gemv_routed_silu_mul: x must be [1, K] and gate_logits [1, num_experts]")
    ne, n, _ = q_weight.shape
    k = x.shape[1]
    if gate_logits.shape[1] != ne:
        raise ValueError(f"moe_gemv_routed_silu_mul: {gate_logits.shape[1]} logits for {ne} experts")
    if n % 2:
        raise ValueError(f"moe_gemv_routed_silu_mul: {n} rows cannot be split into gate and up halves")
    _check_qshapes(q_weight, q_scale, (ne, n), k, bits, group_size)
    out = torch.empty((top_k, n // 2), dtype=x.dtype, device=x.device)
    weights = torch.empty((1, top_k), dtype=x.dtype, device=x.device)
    ids = torch.empty((1, top_k), dtype=torch.int32, device=x.device)
    _lib.call("mi355gq_moe_gemv_routed_silu_mul", x.data_ptr(), gate_logits.data_ptr(), ne, top_k, q_weight.data_ptr(),
              q_scale.data_ptr(), n, k, bits, group_size, _MODEL_DTYPES[x.dtype], weights.data_ptr(), ids.data_ptr(),
              out.data_ptr(), _stream())
    return out, weights, ids


def moe_gemv_combine(x: torch.Tensor, q_weight: torch.Tensor, q_scale: torch.Tensor, expert_ids: torch.Tensor,
                     expert_weights: torch.Tensor, bits: int, group_size: int) -> torch.Tensor:
    """One token: the e2 expert matmul on its top_k rows and the weighted sum over them, in one launch.
    x [top_k, K], expert_ids int32 [1, top_k], expert_weights [1, top_k] (model dtype), q_weight [E, N, nw],
    q_scale [E, N, ng].  Returns out [1, N]; raises Mi355gqError with ERR_UNSUPPORTED where the fused kernel does not
    apply (float32 models, top_k other than 2, short or very long K)."""
    _chk(x, _FLOATS, "x")
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, x.dtype, "q_scale")
    _chk(expert_ids, torch.int32, "expert_ids")
    _chk(expert_weights, x.dtype, "expert_weights")
    if x.dim() != 2 or expert_ids.dim() != 2 or expert_ids.shape[0] != 1 or tuple(expert_weights.shape) != tuple(expert_ids.shape):
        raise ValueError("moe_gemv_combine: x must be [top_k, K], expert_ids and expert_weights [1, top_k]")
    top_k = expert_ids.shape[1]
    if x.shape[0] != top_k:
        raise ValueError(f"moe_gemv_combine: {x.shape[0]} rows of x for {top_k} experts")
    ne, n, _ = q_weight.shape
    k = x.shape[1]
    _check_qshapes(q_weight, q_scale, (ne, n), k, bits, group_size)
    out = torch.empty((1, n), dtype=x.dtype, device=x.device)
    _lib.call("mi355gq_moe_gemv_combine", x.data_ptr(), q_weight.data_ptr(), q_scale.data_ptr(), n, k, bits, group_size,
              _MODEL_DTYPES[x.dtype], ne, expert_ids.data_ptr(), expert_weights.data_ptr(), top_k, out.data_ptr(),
              _stream())
    return out


def moe_gemv(x: torch.Tensor, q_weight: torch.Tensor, q_scale: torch.Tensor,
             expert_ids: torch.Tensor, bits: int, group_size: int, silu_mul_halves: bool = False
             ) -> torch.Tensor:
    """silu_mul_halves: the experts' rows are [gate; up] and the result is silu(gate) * up, [k, N / 2].
    x, q_scale and the result share the model dtype (float16, float32 or bfloat16)."""
    _chk(x, _FLOATS, "x")
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, x.dtype, "q_scale")
    _chk(expert_ids, torch.int32, "expert_ids")
    if x.dim() != 2 or expert_ids.dim() != 2 or expert_ids.shape[0] != 1:
        raise ValueError("moe_gemv: x must be [1|k, K] and expert_ids [1, k]")
    ne, n, _ = q_weight.shape
    k = x.shape[1]
    _check_qshapes(q_weight, q_scale, (ne, n), k, bits, group_size)
    top_k = expert_ids.shape[1]
    if x.dtype != torch.float16:
        dt_args = (x.data_ptr(), x.shape[0], q_weight.data_ptr(), q_scale.data_ptr(), expert_ids.data_ptr(), top_k, ne,
                   n, k, bits, group_size, _MODEL_DTYPES[x.dtype])
        if silu_mul_halves:
            if n % 2:
                raise ValueError(f"moe_gemv: {n} rows cannot be split into gate and up halves")
            out = torch.empty((top_k, n // 2), dtype=x.dtype, device=x.device)
            try:
                _lib.call("mi355gq_moe_gemv_silu_mul_dt", *dt_args, out.data_ptr(), _stream())
                return out
            except _lib.Mi355gqError as err:
                if not _unsupported(err):
                    raise
                return silu_mul(moe_gemv(x, q_weight, q_scale, expert_ids, bits, group_size))
        out = torch.empty((top_k, n), dtype=x.dtype, device=x.device)
        _lib.call("mi355gq_moe_gemv_dt", *dt_args, out.data_ptr(), _stream())
        return out
    args = (x.data_ptr(), x.shape[0], q_weight.data_ptr(), q_scale.data_ptr(), expert_ids.data_ptr(), top_k, ne,
            n, k, bits, group_size)
    if silu_mul_halves:
        if n % 2:
            raise ValueError(f"moe_gemv: {n} rows cannot be split into gate and up halves")
        out = torch.empty((top_k, n // 2), dtype=torch.float16, device=x.device)
        try:
            _lib.call("mi355gq_moe_gemv_silu_mul", *args, out.data_ptr(), _stream())
            return out
        except _lib.Mi355gqError as err:
            if not _unsupported(err):
                raise
            return silu_mul(moe_gemv(x, q_weight, q_scale, expert_ids, bits, group_size))
    out = torch.empty((top_k, n), dtype=torch.float16, device=x.device)
    _lib.call("mi355gq_moe_gemv", *args, out.data_ptr(), _stream())
    return out


def moe_group_gemm(x: torch.Tensor, q_weight: torch.Tensor, q_scale: torch.Tensor,
                   indptr: torch.Tensor, bits: int, group_size: int, silu_mul_halves: bool = False, *, rows_covered: bool = False
                   ) -> torch.Tensor:
    """x, q_scale and the result share the model dtype (float16, float32 or bfloat16).  Rows outside the experts' segments
    come back as zeros; rows_covered: the caller reads no such row, and they are left as they are."""
    new = torch.empty if rows_covered else torch.zeros
    _chk(x, _FLOATS, "x")
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, x.dtype, "q_scale")
    _chk(indptr, (torch.int32, torch.int64), "indptr")
    ne, n, _ = q_weight.shape
    rows, k = x.shape
    _check_qshapes(q_weight, q_scale, (ne, n), k, bits, group_size)
    if tuple(indptr.shape) != (ne + 1,):
        raise ValueError(f"indptr shape {tuple(indptr.shape)}, expected {(ne + 1,)}")
    if x.dtype != torch.float16:
        dt_args = (x.data_ptr(), rows, q_weight.data_ptr(), q_scale.data_ptr(), indptr.data_ptr(),
                   _lib.I64 if indptr.dtype == torch.int64 else _lib.I32, ne, n, k, bits, group_size,
                   _MODEL_DTYPES[x.dtype])
        if silu_mul_halves:
            if n % 2:
                raise ValueError(f"moe_group_gemm: {n} rows cannot be split into gate and up halves")
            out = new((rows, n // 2), dtype=x.dtype, device=x.device)
            try:
                _lib.call("mi355gq_moe_group_gemm_silu_mul_dt", *dt_args, out.data_ptr(), _stream())
                return out
            except _lib.Mi355gqError as err:
                if not _unsupported(err):
                    raise
                return silu_mul(moe_group_gemm(x, q_weight, q_scale, indptr, bits, group_size, rows_covered=rows_covered))
        out = new((rows, n), dtype=x.dtype, device=x.device)
        _lib.call("mi355gq_moe_group_gemm_dt", *dt_args, out.data_ptr(), _stream())
        return out
    args = (x.data_ptr(), rows, q_weight.data_ptr(), q_scale.data_ptr(), indptr.data_ptr(),
            _lib.I64 if indptr.dtype == torch.int64 else _lib.I32, ne, n, k, bits, group_size)
    if silu_mul_halves:
        if n % 2:
            raise ValueError(f"moe_group_gemm: {n} rows cannot be split into gate and up halves")
        out = new((rows, n // 2), dtype=torch.float16, device=x.device)
        try:
            _lib.call("mi355gq_moe_group_gemm_silu_mul", *args, out.data_ptr(), _stream())
            return out
        except _lib.Mi355gqError as err:
            if not _unsupported(err):
                raise
            return silu_mul(moe_group_gemm(x, q_weight, q_scale, indptr, bits, group_size, rows_covered=rows_covered))
    out = new((rows, n), dtype=torch.float16, device=x.device)
    _lib.call("mi355gq_moe_group_gemm", *args, out.data_ptr(), _stream())
    return out


def moe_experts(x: torch.Tensor, x_row_index: Optional[torch.Tensor], q_weight: torch.Tensor,
                q_scale: torch.Tensor, indptr: torch.Tensor, bits: int, group_size: int,
                silu_mul_halves: bool = False, *, rows_covered: bool = False) -> torch.Tensor:
    """moe_group_gemm on x[x_row_index] (the layer's gather folded into the matmul's row addressing);
    x_row_index None: x is already in expert order.  Float16 and bfloat16 models; anything without such a
    kernel (float32 models, odd shapes) runs take_rows and moe_group_gemm."""
    _chk(x, _FLOATS, "x")
    _chk(q_weight, _STORAGE, "q_weight")
    _chk(q_scale, x.dtype, "q_scale")
    _chk(indptr, (torch.int32, torch.int64), "indptr")
    ne, n, _ = q_weight.shape
    x_rows, k = x.shape
    _check_qshapes(q_weight, q_scale, (ne, n), k, bits, group_size)
    if tuple(indptr.shape) != (ne + 1,):
        raise ValueError(f"indptr shape {tuple(indptr.shape)}, expected {(ne + 1,)}")
    rows = x_rows
    if x_row_index is not None:
        _chk(x_row_index, torch.int32, "x_row_index")
        rows = x_row_index.numel()
    if silu_mul_halves and n % 2:
        raise ValueError(f"moe_experts: {n} rows cannot be split into gate and up halves")
    new = torch.empty if rows_covered else torch.zeros
    out = new((rows, n // 2 if silu_mul_halves else n), dtype=x.dtype, device=x.device)
    try:
        _lib.call("mi355gq_moe_experts_dt", x.data_ptr(), x_rows,
                  x_row_index.data_ptr() if x_row_index is not None else None, rows, q_weight.data_ptr(),
                  q_scale.data_ptr(), indptr.data_ptr(), _lib.I64 if indptr.dtype == torch.int64 else _lib.I32,
                  ne, n, k, bits, group_size, _lib.EPILOGUE_SILU_MUL if silu_mul_halves else _lib.EPILOGUE_NONE,
                  _MODEL_DTYPES[x.dtype], out.data_ptr(), _stream())
    except _lib.Mi355gqError as err:
        if not _unsupported(err):
            raise
        gathered = take_rows(x, x_row_index) if x_row_index is not None else x
        return moe_group_gemm(gathered, q_weight, q_scale, indptr, bits, group_size, silu_mul_halves, rows_covered=rows_covered)
    return out


def moe_route(logits: torch.Tensor, top_k: int, indptr_dtype=torch.int32):
    """The routing of a MoE layer in one launch.  Returns (weights [T, k] fp16, ids [T, k] int32,
    token_indices [T * k], reverse_indices [T * k], slot_positions [T * k], indptr [experts + 1]).
    Raises Mi355gqError with code ERR_UNSUPPORTED for batches past the single-workgroup form."""
    _chk(logits, _FLOATS, "logits")
    t, ne = logits.shape
    dev = logits.device
    w = torch.empty((t, top_k), dtype=logits.dtype, device=dev)
    ids = torch.empty((t, top_k), dtype=torch.int32, device=dev)
    tok, rev, pos = (torch.empty((t * top_k,), dtype=torch.int32, device=dev) for _ in range(3))
    indptr = torch.empty((ne + 1,), dtype=indptr_dtype, device=dev)
    _lib.call("mi355gq_moe_route_dt", logits.data_ptr(), t, ne, top_k, w.data_ptr(), ids.data_ptr(), tok.data_ptr(),
              rev.data_ptr(), pos.data_ptr(), indptr.data_ptr(),
              _lib.I64 if indptr_dtype == torch.int64 else _lib.I32, _MODEL_DTYPES[logits.dtype], _stream())
    return w, ids, tok, rev, pos, indptr


def moe_combine_sorted(y: torch.Tensor, slot_positions: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
    """y fp16 [T * k, H] in expert-sorted order, slot_positions int32 [T * k], weights fp16 [T, k] -> [T, H]."""
    _chk(y, _FLOATS, "y")
    _chk(slot_positions, torch.int32, "slot_positions")
    _chk(weights, y.dtype, "weights")
    t, k = weights.shape
    if y.shape[0] != t * k or slot_positions.numel() != t * k:
        raise ValueError("moe_combine_sorted: y and slot_positions must have T * k rows")
    h = y.shape[1]
    out = torch.empty((t, h), dtype=y.dtype, device=y.device)
    _lib.call("mi355gq_moe_combine_dt", y.data_ptr(), slot_positions.data_ptr(), weights.data_ptr(), t, k, h,
              out.data_ptr(), _MODEL_DTYPES[y.dtype], _stream())
    return out


def gating_softmax_topk(logits: torch.Tensor, top_k: int, norm_topk_prob: bool = True
                        ) -> Tuple[torch.Tensor, torch.Tensor]:
    _chk(logits, _FLOATS, "logits")
    t, ne = logits.shape
    w = torch.empty((t, top_k), dtype=logits.dtype, device=logits.device)
    ids = torch.empty((t, top_k), dtype=torch.int32, device=logits.device)
    _lib.call("mi355gq_gating_softmax_topk_ex", logits.data_ptr(), t, ne, top_k, 1 if norm_topk_prob else 0,
              _MODEL_DTYPES[logits.dtype], w.data_ptr(), ids.data_ptr(), _stream())
    return w, ids


def gating_topk(scores: torch.Tensor, top_k: int) -> Tuple[torch.Tensor, torch.Tensor]:
    _chk(scores, _FLOATS, "scores")
    t, ne = scores.shape
    w = torch.empty((t, top_k), dtype=scores.dtype, device=scores.device)
    ids = torch.empty((t, top_k), dtype=torch.int32, device=scores.device)
    _lib.call("mi355gq_gating_topk", scores.data_ptr(), t, ne, top_k, w.data_ptr(), ids.data_ptr(),
              _MODEL_DTYPES[scores.dtype], _stream())
    return w, ids


def moe_cumsum(expert_indices: torch.Tensor, num_local_experts: int) -> torch.Tensor:
    _chk(expert_indices, torch.int32, "expert_indices")
    t, k = expert_indices.shape
    out = torch.empty((num_local_experts * t,), dtype=torch.int32, device=expert_indices.device)
    _lib.call("mi355gq_moe_cumsum", expert_indices.data_ptr(), t, k, num_local_experts,
              out.data_ptr(), _stream())
    return out


def get_indices(cumsum: torch.Tensor, expert_indices: torch.Tensor
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    _chk(cumsum, torch.int32, "cumsum")
    _chk(expert_indices, torch.int32, "expert_indices")
    t, k = expert_indices.shape
    ne = cumsum.numel() // t if t else 1
    rev = torch.zeros((t * k,), dtype=torch.int32, device=cumsum.device)
    tok = torch.zeros((t * k,), dtype=torch.int32, device=cumsum.device)
    _lib.call("mi355gq_moe_get_indices", cumsum.data_ptr(), expert_indices.data_ptr(), t, k, ne,
              rev.data_ptr(), tok.data_ptr(), _stream())
    return rev, tok


def get_indptr(cumsum: torch.Tensor, num_local_experts: int, batch_size: int, inclusive: bool,
               out_dtype=torch.int32) -> torch.Tensor:
    _chk(cumsum, torch.int32, "cumsum")
    n = num_local_experts if inclusive else num_local_experts + 1
    out = torch.empty((n,), dtype=out_dtype, device=cumsum.device)
    _lib.call("mi355gq_moe_get_indptr", cumsum.data_ptr(), num_local_experts, batch_size,
              int(inclusive), _lib.I64 if out_dtype == torch.int64 else _lib.I32, out.data_ptr(),
              _stream())
    return out


def take_rows(x: torch.Tensor, indices: torch.Tensor, *, rows_covered: bool = False) -> torch.Tensor:
    """x[indices]; an index outside x gives a row of zeros (rows_covered: a row that is left as it is and that the caller
    does not read)."""
    _chk(x, _FLOATS, "x")
    _chk(indices, torch.int32, "indices")
    r, h = indices.numel(), x.shape[1]
    out = (torch.empty if rows_covered else torch.zeros)((r, h), dtype=x.dtype, device=x.device)
    _lib.call("mi355gq_take_rows_dt", x.data_ptr(), indices.data_ptr(), r, h, x.shape[0],
              out.data_ptr(), _MODEL_DTYPES[x.dtype], _stream())
    return out


def scatter_output(x: torch.Tensor, indices: torch.Tensor) -> torch.Tensor:
    _chk(x, _FLOATS, "x")
    _chk(indices, torch.int32, "indices")
    r, h = x.shape
    out = torch.zeros_like(x)
    _lib.call("mi355gq_moe_scatter_output_dt", x.data_ptr(), indices.data_ptr(), r, h,
              out.data_ptr(), _MODEL_DTYPES[x.dtype], _stream())
    return out


def silu_mul(x: torch.Tensor) -> torch.Tensor:
    _chk(x, _FLOATS, "x")
    r, two_i = x.shape
    out = torch.empty((r, two_i // 2), dtype=x.dtype, device=x.device)
    _lib.call("mi355gq_silu_mul_dt", x.data_ptr(), r, two_i // 2, out.data_ptr(), _MODEL_DTYPES[x.dtype], _stream())
    return out


def moe_combine(y: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
    """y [T, k, H], weights [T, k] -> [T, H], all in the model dtype."""
    _chk(y, _FLOATS, "y")
    _chk(weights, y.dtype, "weights")
    t, k, h = y.shape
    out = torch.empty((t, h), dtype=y.dtype, device=y.device)
    _lib.call("mi355gq_moe_combine_dt", y.data_ptr(), None, weights.data_ptr(), t, k, h, out.data_ptr(),
              _MODEL_DTYPES[y.dtype], _stream())
    return out


# ---- 8-bit block-scaled models ----
#
# An e4m3 tensor is a torch.float8_e4m3fn tensor whose rows lie a multiple of 16 bytes apart (its last dimension contiguous; rows
# of a last size that is no multiple of 16 are a view of a wider allocation, as fp8_quantize and fp8_quantize_weight make them).

FP8_BLOCK = 128
_E4M3 = torch.float8_e4m3fn
_SCORING = {"softmax": _lib.SCORE_SOFTMAX, "sigmoid": _lib.SCORE_SIGMOID}


def _fp8_empty(lead, k: int, device) -> torch.Tensor:
    return torch.empty((*lead, -(-k // 16) * 16), dtype=_E4M3, device=device)[..., :k]


def _chk_fp8(t: torch.Tensor, name: str, dims: int) -> int:
    """The pitch of an e4m3 tensor's rows in bytes."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name}: must live on the GPU (got {t.device})")
    if t.dtype != _E4M3:
        raise TypeError(f"{name}: dtype {t.dtype}, expected {_E4M3}")
    if t.dim() != dims:
        raise ValueError(f"{name}: {t.dim()} dimensions, expected {dims}")
    n, k = t.shape[-2:]
    row = -(-k // 16) * 16  # what the kernels' loads touch of one
    if n > 1:
        pitch = t.stride(-2)
    else:  # (of a single row the stride says nothing)
        pitch = t.stride(0) if dims == 3 and t.shape[0] > 1 else row
    if t.numel() and ((k > 1 and t.stride(-1) != 1) or pitch < k or pitch % 16
                      or (dims == 3 and t.shape[0] > 1 and t.stride(0) != n * pitch)):
        raise ValueError(f"{name}: rows must be contiguous and lie a multiple of 16 bytes apart (strides {t.stride()}); "
                         "fp8_quantize_weight makes such a tensor, torch.nn.functional.pad one of a checkpoint's")
    if t.numel() and t.untyped_storage().nbytes() - t.storage_offset() < (t.numel() // k - 1) * pitch + row:
        raise ValueError(f"{name}: the last row of {k} bytes needs {row} of storage")
    return max(pitch, row)


def _chk_scale(t: torch.Tensor, shape, name: str) -> torch.Tensor:
    _chk(t, torch.float32, name)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def fp8_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [rows, K] -> e4m3 [rows, K] in groups of 128 along K, and their scales float32 [ceil(K / 128), rows]: the smallest
    power of two that brings a group's largest magnitude to 448 or below."""
    native = _lib.native()
    done = native.fp8_quantize(x) if native is not None else None
    if isinstance(done, tuple):
        return done
    if done is not None:
        raise _lib.failed("mi355gq_fp8_quantize", done)
    _chk(x, _FLOATS, "x")
    if x.dim() != 2:
        raise ValueError(f"fp8_quantize: x must be [rows, K], got {tuple(x.shape)}")
    rows, k = x.shape
    q = _fp8_empty((rows,), k, x.device)
    scale = torch.empty((-(-k // FP8_BLOCK), rows), dtype=torch.float32, device=x.device)
    _lib.call("mi355gq_fp8_quantize", x.data_ptr(), rows, k, _MODEL_DTYPES[x.dtype], q.data_ptr(), -(-k // 16) * 16, scale.data_ptr(),
              _stream())
    return q, scale


def fp8_silu_mul_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp8_quantize of silu(x1) * x2, x [rows, 2 K] = [x1, x2], computed in float32."""
    _chk(x, _FLOATS, "x")
    if x.dim() != 2 or x.shape[1] % 2:
        raise ValueError(f"fp8_silu_mul_quantize: x must be [rows, 2 K], got {tuple(x.shape)}")
    rows, k = x.shape[0], x.shape[1] // 2
    q = _fp8_empty((rows,), k, x.device)
    scale = torch.empty((-(-k // FP8_BLOCK), rows), dtype=torch.float32, device=x.device)
    _lib.call("mi355gq_fp8_silu_mul_quantize", x.data_ptr(), rows, k, _MODEL_DTYPES[x.dtype], q.data_ptr(), -(-k // 16) * 16,
              scale.data_ptr(), _stream())
    return q, scale


def fp8_quantize_weight(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """w [..., N, K] -> e4m3 [..., N, K] and a scale for each block of 128 x 128, float32 [..., ceil(N / 128), ceil(K / 128)]."""
    _chk(w, _FLOATS, "w")
    if w.dim() not in (2, 3):
        raise ValueError(f"fp8_quantize_weight: w must be [N, K] or [experts, N, K], got {tuple(w.shape)}")
    lead, (n, k) = tuple(w.shape[:-2]), w.shape[-2:]
    q = _fp8_empty((*lead, n), k, w.device)
    scale = torch.empty((*lead, -(-n // FP8_BLOCK), -(-k // FP8_BLOCK)), dtype=torch.float32, device=w.device)
    _lib.call("mi355gq_fp8_quantize_weight", w.data_ptr(), lead[0] if lead else 1, n, k, _MODEL_DTYPES[w.dtype], q.data_ptr(),
              -(-k // 16) * 16, scale.data_ptr(), _stream())
    return q, scale


def fp8_dequantize(q: torch.Tensor, scale: torch.Tensor, out_dtype=torch.float32, row_groups: bool = False) -> torch.Tensor:
    """q * scale of e4m3 weights [..., N, K] with their block scales, or (row_groups) of activations [rows, K] with theirs."""
    pitch = _chk_fp8(q, "q", 2 if row_groups else q.dim() if isinstance(q, torch.Tensor) and q.dim() == 3 else 2)
    lead, (n, k) = tuple(q.shape[:-2]), q.shape[-2:]
    groups = -(-k // FP8_BLOCK)
    _chk_scale(scale, (groups, n) if row_groups else (*lead, -(-n // FP8_BLOCK), groups), "scale")
    if out_dtype not in _MODEL_DTYPES:
        raise TypeError(f"out_dtype {out_dtype}")
    out = torch.empty(q.shape, dtype=out_dtype, device=q.device)
    _lib.call("mi355gq_fp8_dequantize", q.data_ptr(), pitch, scale.data_ptr(), lead[0] if lead else 1, n, k, 1 if row_groups else 0,
              _MODEL_DTYPES[out_dtype], out.data_ptr(), _stream())
    return out


def fp8_linear(x, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, out_dtype=None,
               residual: Optional[torch.Tensor] = None, precise: Optional[bool] = None) -> torch.Tensor:
    """y[..., N] = x[..., K] . (weight * weight_scale)^T (+ bias) (+ residual), both operands in e4m3.

    x: a float16, bfloat16 or float32 tensor, which is quantised on the way as fp8_quantize does, or the pair (q, scale) that
    fp8_quantize gives.  weight e4m3 [N, K], weight_scale float32 [ceil(N / 128), ceil(K / 128)].  bias and residual have x's
    type (of a pair: the output's, float16 by default), the output out_dtype, or that type.

    precise: blocks of 128 are summed in float32.  Without it they may be summed by the 8-bit matrix instructions, which of eight
    neighbouring products drop what lies more than 13 bits below the largest: 1.5e-5 of a whole result's norm for normal x and weights, 8e-5
    where channels of x differ by factors of seven; more of a single result that is far below its products.  None: a float32 output is
    precise, a 16-bit one (whose rounding is 2e-4 in float16, 1.7e-3 in bfloat16) is not.  Blocks join one another in float32 either way."""
    native = _lib.native()
    done = native.fp8_linear(x, weight, weight_scale, bias, out_dtype, residual, precise) if native is not None else None
    if isinstance(done, torch.Tensor):
        return done
    if done is not None:
        raise _lib.failed("mi355gq_fp8_linear", done)
    pair = isinstance(x, (tuple, list))
    if pair:
        if len(x) != 2:
            raise ValueError("fp8_linear: x must be a tensor or the pair (q, scale)")
        q, x_scale = x
        x_pitch = _chk_fp8(q, "x", 2)
        _chk_scale(x_scale, (-(-q.shape[1] // FP8_BLOCK), q.shape[0]), "x scale")
        out_dtype = torch.float16 if out_dtype is None else out_dtype
        dtype, x = out_dtype, q
    else:
        _chk(x, _FLOATS, "x")
        x_scale, x_pitch, dtype = None, 0, x.dtype
        out_dtype = dtype if out_dtype is None else out_dtype
    if out_dtype not in _MODEL_DTYPES:
        raise TypeError(f"out_dtype {out_dtype}")
    w_pitch = _chk_fp8(weight, "weight", 2)
    n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k or k == 0:
        raise ValueError(f"fp8_linear: x {tuple(x.shape)} for a weight of {tuple(weight.shape)}")
    _chk_scale(weight_scale, (-(-n // FP8_BLOCK), -(-k // FP8_BLOCK)), "weight_scale")
    m = 1
    for d in x.shape[:-1]:
        m *= d
    shape = (*x.shape[:-1], n)
    if bias is not None:
        _chk(bias, dtype, "bias")
        if tuple(bias.shape) != (n,):
            raise ValueError(f"bias shape {tuple(bias.shape)}, expected {(n,)}")
    if residual is not None:
        _chk(residual, dtype, "residual")
        if tuple(residual.shape) != shape:
            raise ValueError(f"residual shape {tuple(residual.shape)}, expected {shape}")
    out = torch.empty(shape, dtype=out_dtype, device=x.device)
    ws_bytes = _lib.lib().mi355gq_fp8_linear_workspace_bytes(m, n, k, 1 if pair else 0)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    _lib.call("mi355gq_fp8_linear", x.data_ptr(), x_pitch, x_scale.data_ptr() if pair else None, weight.data_ptr(), w_pitch,
              weight_scale.data_ptr(), bias.data_ptr() if bias is not None else None,
              residual.data_ptr() if residual is not None else None, m, n, k, _MODEL_DTYPES[dtype], _MODEL_DTYPES[out_dtype],
              1 if (out_dtype == torch.float32 if precise is None else precise) else 0, out.data_ptr(), ws.data_ptr() if ws is not None else None, ws_bytes, _stream())
    return out


def fp8_group_gemm(q: torch.Tensor, scale: torch.Tensor, x_row_index: Optional[torch.Tensor], weight: torch.Tensor,
                   weight_scale: torch.Tensor, indptr: torch.Tensor, out_dtype=torch.float16, precise: Optional[bool] = None
                   ) -> torch.Tensor:
    """The product by expert segments: y[r] = x[x_row_index[r]] . weight[e]^T for indptr[e] <= r < indptr[e + 1]; q, scale as
    fp8_quantize gives them, weight e4m3 [experts, N, K].  x_row_index None: row r of x.  Rows outside every segment are zeros.
    precise: see fp8_linear."""
    x_pitch, w_pitch = _chk_fp8(q, "q", 2), _chk_fp8(weight, "weight", 3)
    experts, n, k = weight.shape
    if q.shape[1] != k or k == 0:
        raise ValueError(f"fp8_group_gemm: q {tuple(q.shape)} for weights of {tuple(weight.shape)}")
    groups = -(-k // FP8_BLOCK)
    _chk_scale(scale, (groups, q.shape[0]), "scale")
    _chk_scale(weight_scale, (experts, -(-n // FP8_BLOCK), groups), "weight_scale")
    _chk(indptr, torch.int32, "indptr")
    if tuple(indptr.shape) != (experts + 1,):
        raise ValueError(f"indptr shape {tuple(indptr.shape)}, expected {(experts + 1,)}")
    if out_dtype not in _MODEL_DTYPES:
        raise TypeError(f"out_dtype {out_dtype}")
    rows = q.shape[0]
    if x_row_index is not None:
        _chk(x_row_index, torch.int32, "x_row_index")
        rows = x_row_index.numel()
    out = torch.zeros((rows, n), dtype=out_dtype, device=q.device)
    _lib.call("mi355gq_fp8_group_gemm", q.data_ptr(), x_pitch, scale.data_ptr(), q.shape[0],
              x_row_index.data_ptr() if x_row_index is not None else None, rows, weight.data_ptr(), w_pitch, weight_scale.data_ptr(),
              indptr.data_ptr(), experts, n, k, _MODEL_DTYPES[out_dtype],
              1 if (out_dtype == torch.float32 if precise is None else precise) else 0, out.data_ptr(), _stream())
    return out


def moe_gating(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, num_groups: int = 1,
               top_groups: int = 1, renormalize: bool = True, scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Router logits [T, experts] -> (weights float32 [T, top_k], ids int32 [T, top_k]), best first.

    scoring: "softmax" over the row, or "sigmoid" of each logit.  bias float32 [experts] is added for the choice, not to the
    weights.  num_groups > 1: only the experts of the top_groups best of that many equal runs of experts are chosen from; a
    run stands by its best key, or with a bias by the sum of its two best.  renormalize: the chosen scores are divided by their
    sum.  Ties keep the lower index; a NaN logit is chosen last."""
    native = _lib.native()
    done = native.moe_gating(logits, top_k, scoring, bias, num_groups, top_groups, renormalize, scale) if native is not None else None
    if isinstance(done, tuple):
        return done
    if done is not None:
        raise _lib.failed("mi355gq_moe_gating", done)
    _chk(logits, _FLOATS, "logits")
    if logits.dim() != 2:
        raise ValueError(f"moe_gating: logits must be [T, experts], got {tuple(logits.shape)}")
    if scoring not in _SCORING:
        raise ValueError(f"moe_gating: scoring {scoring!r}, expected one of {sorted(_SCORING)}")
    t, ne = logits.shape
    if bias is not None:
        _chk_scale(bias, (ne,), "bias")
    weights = torch.empty((t, max(top_k, 0)), dtype=torch.float32, device=logits.device)
    ids = torch.empty((t, max(top_k, 0)), dtype=torch.int32, device=logits.device)
    _lib.call("mi355gq_moe_gating", logits.data_ptr(), bias.data_ptr() if bias is not None else None, t, ne, top_k, _SCORING[scoring],
              num_groups, top_groups, 1 if renormalize else 0, float(scale), _MODEL_DTYPES[logits.dtype], weights.data_ptr(),
              ids.data_ptr(), _stream())
    return weights, ids


def moe_plan(ids: torch.Tensor, num_experts: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """ids int32 [T, k] -> the slots in the order of their expert: (row_token [T * k], slot_row [T * k], indptr [experts + 1])."""
    _chk(ids, torch.int32, "ids")
    if ids.dim() != 2:
        raise ValueError(f"moe_plan: ids must be [T, k], got {tuple(ids.shape)}")
    t, k = ids.shape
    row_token, slot_row = (torch.zeros((t * k,), dtype=torch.int32, device=ids.device) for _ in range(2))
    indptr = torch.empty((max(num_experts, 0) + 1,), dtype=torch.int32, device=ids.device)
    _lib.call("mi355gq_moe_plan", ids.data_ptr(), t, k, num_experts, row_token.data_ptr(), slot_row.data_ptr(), indptr.data_ptr(),
              _stream())
    return row_token, slot_row, indptr


def fp8_moe_experts(x: torch.Tensor, weights: torch.Tensor, ids: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor,
                    w2: torch.Tensor, w2_scale: torch.Tensor) -> torch.Tensor:
    """One expert layer on routed tokens: x [T, hidden] float16 or bfloat16, weights float32 [T, k] and ids int32 [T, k] as
    moe_gating gives them, w13 e4m3 [experts, 2 inter, hidden] (gate rows, then up rows), w2 e4m3 [experts, hidden, inter].
    An id outside the experts adds nothing.  A block of w13's scales that holds both gate and up rows, where inter is no multiple of 128, is of both.

    Gate and up are summed in float32, the second product as fp8_linear does for a 16-bit output; moe_plan, fp8_quantize, fp8_group_gemm
    with precise and fp8_silu_mul_quantize are the same layer in steps, in float32 throughout."""
    _chk(x, (torch.float16, torch.bfloat16), "x")
    _chk(ids, torch.int32, "ids")
    pitch13, pitch2 = _chk_fp8(w13, "w13", 3), _chk_fp8(w2, "w2", 3)
    ne, hidden, inter = w2.shape
    if tuple(w13.shape) != (ne, 2 * inter, hidden) or x.dim() != 2 or x.shape[1] != hidden:
        raise ValueError(f"fp8_moe: x {tuple(x.shape)}, w13 {tuple(w13.shape)} and w2 {tuple(w2.shape)} do not belong together")
    t = x.shape[0]
    if ids.dim() != 2 or ids.shape[0] != t:
        raise ValueError(f"fp8_moe: ids {tuple(ids.shape)} for {t} tokens")
    _chk_scale(weights, ids.shape, "weights")
    _chk_scale(w13_scale, (ne, -(-2 * inter // FP8_BLOCK), -(-hidden // FP8_BLOCK)), "w13_scale")
    _chk_scale(w2_scale, (ne, -(-hidden // FP8_BLOCK), -(-inter // FP8_BLOCK)), "w2_scale")
    k = ids.shape[1]
    if x.data_ptr() % 16:  # the quantiser's loads
        x = x.clone()
    out = torch.empty_like(x)
    ws_bytes = _lib.lib().mi355gq_fp8_moe_workspace_bytes(t, hidden, inter, ne, k)
    if ws_bytes and 2 * inter * pitch13 >= 2**32 - 1:
        ws_bytes += 8 * t * k * inter + 256
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    _lib.call("mi355gq_fp8_moe", x.data_ptr(), t, hidden, inter, ne, k, weights.data_ptr(), ids.data_ptr(), w13.data_ptr(), pitch13,
              w13_scale.data_ptr(), w2.data_ptr(), pitch2, w2_scale.data_ptr(), _MODEL_DTYPES[x.dtype], out.data_ptr(),
              ws.data_ptr() if ws is not None else None, ws_bytes, _stream())
    return out


def fp8_moe(x: torch.Tensor, logits: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor,
            w2_scale: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, num_groups: int = 1,
            top_groups: int = 1, renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """moe_gating on the router's logits [T, experts], then fp8_moe_experts."""
    native = _lib.native()
    done = None
    if native is not None:
        done = native.fp8_moe(x, w13, w13_scale, w2, w2_scale, logits, top_k, scoring, bias, num_groups, top_groups, renormalize, scale)
    if done is not None:
        return done
    weights, ids = moe_gating(logits, top_k, scoring, bias, num_groups, top_groups, renormalize, scale)
    return fp8_moe_experts(x, weights, ids, w13, w13_scale, w2, w2_scale)
