"""Grouped-GEMM stage of the per-channel W8A8 MoE (reference: lightop.gemmopt.moe_gemm_w8a8, python/lightop/gemmopt.py:437-457;
native side csrc/moe_gemm/w8a8/moe_w8a8.cu:2389-2536), and the dense products beside it: e4m3 with block scales, 16-bit and int8 with
bias, activation and residual in their epilogue or both projections of a gated block in one."""
from __future__ import annotations

from typing import Any, Dict, Optional

import torch

from . import _lib
from .op import _act_dtype, _on_device, _one_device, _require_cuda, _rows16, _strided_rows


_OUT_DTYPES = {torch.bfloat16: _lib.LO_BF16, torch.float16: _lib.LO_F16, torch.float32: _lib.LO_F32}


def moe_gemm_w8a8(input: torch.Tensor, b_qweight: torch.Tensor, output: torch.Tensor, a_scale: torch.Tensor,
                  b_scale: torch.Tensor, topk_weights: Optional[torch.Tensor], sorted_token_ids: torch.Tensor,
                  experts_ids: torch.Tensor, num_tokens_post_pad: torch.Tensor, top_k: int,
                  config: Dict[str, Any], flags: int = 0, global_num_experts: int = 0) -> torch.Tensor:
    """One grouped GEMM stage in the per-channel form (reference: moe_gemm_w8a8, gemmopt.py:437-457):
    output[f] = T((sum_k input[f // top_k] * b_qweight[e]) * ts * b_scale[e]) with
    ts = a_scale[f // top_k], times topk_weights[f] when they are given (the second stage).
    ``a_scale`` [rows(, 1)], ``b_scale`` [E, N(, 1)]; ``config`` needs ``BLOCK_SIZE_M`` (the reference's
    ``MODE`` / ``DELTA`` pick among its tuned kernels and are ignored)."""
    _require_cuda(input, b_qweight, output, a_scale, b_scale, topk_weights, sorted_token_ids, experts_ids,
                  num_tokens_post_pad)
    assert input.dtype == torch.int8 and b_qweight.dtype == torch.int8
    assert input.is_contiguous() and b_qweight.is_contiguous() and output.is_contiguous()
    E, N, K = b_qweight.shape
    assert input.shape[1] == K and output.shape[-1] == N
    assert a_scale.dtype == torch.float32 and a_scale.is_contiguous() and a_scale.numel() == input.shape[0]
    assert b_scale.dtype == torch.float32 and b_scale.is_contiguous() and b_scale.numel() == E * N
    assert sorted_token_ids.dtype == torch.int32 and experts_ids.dtype == torch.int32
    num_valid = output.numel() // N
    tw = None
    if topk_weights is not None:
        tw = topk_weights if topk_weights.dtype == torch.float32 and topk_weights.is_contiguous() \
            else topk_weights.to(torch.float32).contiguous()
    with _on_device(input):
        _lib.check(_lib.lib().lo_moe_gemm_w8a8(
            _lib.ptr(input), _lib.ptr(a_scale), _lib.ptr(b_qweight), _lib.ptr(b_scale), _lib.ptr(output),
            _act_dtype(output), _lib.ptr(tw), _lib.ptr(sorted_token_ids), _lib.ptr(experts_ids),
            _lib.ptr(num_tokens_post_pad), sorted_token_ids.numel(), num_valid, input.shape[0], E,
            int(global_num_experts or 0), N, K, int(top_k),
            int(config["BLOCK_SIZE_M"]), 1 if tw is not None else 0,
            flags | (_lib.LO_GEMM_W_PRESHUFFLED if bool(getattr(b_qweight, "lo_preshuffled", False)) else 0), _lib.stream_of(input)))
    return output


def gemm_w8a8_fp8_block(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor,
                        out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Dense product of e4m3 operands with block scales, as a shared expert or a projection of an fp8 checkpoint needs:
    ``out[m, n] = sum_kb (a[m, kb] . b[n, kb]) * a_scale[m, kb] * b_scale[n // 128, kb]`` over K blocks of 128, summed in fp32
    and rounded once to ``out_dtype`` (bfloat16, float16 or float32).

    ``a`` [..., K] with ``a_scale`` [..., K/128] (``per_token_group_quant_fp8``), ``b`` [N, K] row-major as a checkpoint holds it,
    ``b_scale`` [ceil(N/128), K/128] fp32; any number of rows, any N, K a multiple of 128.  Written into ``out`` (contiguous)
    where the caller brings it."""
    if out is None:
        made = (_lib._host or _lib.host()).gemm_fp8(a, b, a_scale, b_scale, _OUT_DTYPES.get(out_dtype, -1))
        if made is not None:
            return made
    _one_device(a, b, a_scale, b_scale, out)
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn:
        raise RuntimeError(f"gemm_w8a8_fp8_block: a and b must be float8_e4m3fn, got {a.dtype} and {b.dtype}")
    if a.dim() < 1 or b.dim() != 2 or a.shape[-1] != b.shape[1]:
        raise RuntimeError(f"gemm_w8a8_fp8_block: a must be [..., K] and b [N, K], got {tuple(a.shape)} and {tuple(b.shape)}")
    N, K = b.shape
    if K == 0 or K % 128:
        raise RuntimeError(f"gemm_w8a8_fp8_block: K must be a multiple of 128, got {K}")
    if a_scale.shape != a.shape[:-1] + (K // 128,) or b_scale.shape != ((N + 127) // 128, K // 128):
        raise RuntimeError("gemm_w8a8_fp8_block: scales must be [..., K/128] and [ceil(N/128), K/128], got "
                           f"{tuple(a_scale.shape)} and {tuple(b_scale.shape)}")
    if a_scale.dtype != torch.float32 or b_scale.dtype != torch.float32:
        raise RuntimeError("gemm_w8a8_fp8_block: scales must be float32")
    shape = a.shape[:-1] + (N,)
    if out_dtype not in _OUT_DTYPES:
        raise RuntimeError(f"gemm_w8a8_fp8_block: out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=a.device)
    elif out.shape != shape or out.dtype != out_dtype or not out.is_contiguous():
        raise RuntimeError(f"gemm_w8a8_fp8_block: out must be a contiguous {out_dtype} tensor of shape {tuple(shape)}")
    dtype = _OUT_DTYPES[out_dtype]
    if out.numel() == 0:
        return out
    from .moe import native  # (which imports this module)

    a, b, a_scale, b_scale = _rows16(a), _rows16(b), a_scale.contiguous(), b_scale.contiguous()
    lib, M = _lib.lib(), out.numel() // N
    nbytes = lib.lo_gemm_w8a8_fp8_block_workspace_bytes(M, N, K, dtype)
    _lib.check(nbytes)
    with _on_device(a):
        stream = torch.cuda.current_stream(a.device).cuda_stream
        scratch = native._scratch(nbytes, a.device, stream) if nbytes else None
        _lib.check(lib.lo_gemm_w8a8_fp8_block(_lib.ptr(a), _lib.ptr(a_scale), _lib.ptr(b), _lib.ptr(b_scale), _lib.ptr(out), dtype, M, N, K,
                                              _lib.ptr(scratch), nbytes, _lib.stream_of(a)))
    return out


_ACTIVATIONS = {None: _lib.LO_ACT_NONE, "silu": _lib.LO_ACT_SILU, "gelu": _lib.LO_ACT_GELU}
_OPERANDS = {torch.bfloat16: _lib.LO_BF16, torch.float16: _lib.LO_F16, torch.int8: _lib.LO_I8}
_MOST_STRIDE = 4 << 20  # bytes from one row to the next that the kernels take


def _operand(t: torch.Tensor) -> torch.Tensor:
    """An operand as rows that the kernels take: a view where it can be."""
    t = _strided_rows(t)
    return t if t.shape[0] <= 1 or t.stride(0) * t.element_size() <= _MOST_STRIDE else t.contiguous()


def _dense(name: str, a, b, a_scale, b_scale, bias, activation, gated: bool, scale: float, residual, out_dtype, out) -> torch.Tensor:
    if activation not in _ACTIVATIONS or (gated and activation is None):
        raise ValueError(f"{name}: unsupported activation {activation!r}")
    made = (_lib._host or _lib.host()).gemm_dense(a, b, a_scale, b_scale, bias, residual, out, _ACTIVATIONS[activation], gated, scale,
                                                  _OUT_DTYPES.get(out_dtype, -1))
    if made is not None:
        return made
    _one_device(a, b, a_scale, b_scale, bias, residual, out)
    int8 = a_scale is not None
    if a.dtype != b.dtype or (a.dtype != torch.int8 if int8 else a.dtype not in (torch.bfloat16, torch.float16)):
        raise RuntimeError(f"{name}: a and b must both be {'int8' if int8 else 'bfloat16 or float16'}, got {a.dtype} and {b.dtype}")
    if a.dim() < 1 or b.dim() != 2 or a.shape[-1] != b.shape[1]:
        raise RuntimeError(f"{name}: a must be [..., K] and b [{'2 N' if gated else 'N'}, K], got {tuple(a.shape)} and {tuple(b.shape)}")
    rows, K = b.shape
    unit = 16 if int8 else 8
    if K == 0 or K % unit:
        raise RuntimeError(f"{name}: K must be a multiple of {unit}, got {K}")
    if gated and rows % 2:
        raise RuntimeError(f"{name}: b must hold as many rows of the gate as of the other projection, got {rows}")
    N = rows // 2 if gated else rows
    M = a.numel() // K
    if int8 and (a_scale.shape not in (a.shape[:-1], a.shape[:-1] + (1,)) or b_scale.shape not in ((rows,), (rows, 1))
                 or a_scale.dtype != torch.float32 or b_scale.dtype != torch.float32):
        raise RuntimeError(f"{name}: scales must be float32, one for a row: {tuple(a.shape[:-1])} and ({rows},), got "
                           f"{tuple(a_scale.shape)} {a_scale.dtype} and {tuple(b_scale.shape)} {b_scale.dtype}")
    if out_dtype not in _OUT_DTYPES:
        raise RuntimeError(f"{name}: out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    if bias is not None and (bias.shape != (rows,) or bias.dtype not in (out_dtype, torch.float32)):
        raise RuntimeError(f"{name}: bias must be [{rows}], {out_dtype} or float32, got {tuple(bias.shape)} {bias.dtype}")
    shape = a.shape[:-1] + (N,)
    if residual is not None and (residual.shape != shape or residual.dtype != out_dtype):
        raise RuntimeError(f"{name}: residual must be {tuple(shape)} {out_dtype}, got {tuple(residual.shape)} {residual.dtype}")
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=a.device)
    elif out.shape != shape or out.dtype != out_dtype or not out.is_contiguous():
        raise RuntimeError(f"{name}: out must be a contiguous {out_dtype} tensor of shape {tuple(shape)}")
    if out.numel() == 0:
        return out
    from .moe import native  # (which imports this module)

    operands, kind, result = [_operand(t) for t in (a, b)], _OPERANDS[a.dtype], _OUT_DTYPES[out_dtype]
    if int8:
        a_scale, b_scale = a_scale.contiguous(), b_scale.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    if residual is not None:
        residual = residual.reshape(M, N)
        if N > 1 and residual.stride(1) != 1 or M > 1 and residual.stride(0) < N:
            residual = residual.contiguous()
    lib = _lib.lib()
    nbytes = lib.lo_gemm_bias_act_workspace_bytes(kind, int(gated), M, N, K)
    _lib.check(nbytes)
    with _on_device(a):
        stream = torch.cuda.current_stream(a.device).cuda_stream
        scratch = native._scratch(nbytes, a.device, stream) if nbytes else None
        _lib.check(lib.lo_gemm_bias_act(
            _lib.ptr(operands[0]), operands[0].stride(0), _lib.ptr(operands[1]), operands[1].stride(0), kind, _lib.ptr(a_scale), _lib.ptr(b_scale),
            _lib.ptr(bias), result if bias is None else _OUT_DTYPES[bias.dtype], _ACTIVATIONS[activation], int(gated), float(scale),
            _lib.ptr(residual), 0 if residual is None else residual.stride(0), _lib.ptr(out), result, M, N, K, _lib.ptr(scratch), nbytes,
            _lib.stream_of(a)))
    return out


def gemm_bias_act(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                  residual: Optional[torch.Tensor] = None, scale: float = 1.0, out_dtype: Optional[torch.dtype] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Dense product with its epilogue, for what a quantised checkpoint keeps in 16 bits (a router, projections, the
    vocabulary's): ``out = scale * act(a b^T + bias) + residual``, summed and finished in fp32 and rounded once to ``out_dtype``
    (bfloat16, float16 or float32; a's type by default).

    ``a`` [..., K] and ``b`` [N, K] both bfloat16 or both float16, row-major (rows may be strided), any number of rows and any N up to
    2^24 and 2^23 (and 2^22 tiles of 256 x 256 results), K a multiple of 8 up to 2097152; ``bias`` [N] of ``out_dtype`` or float32; ``activation`` None, "silu" or "gelu" (its erf form); ``residual`` [..., N] of
    ``out_dtype``.  Written into ``out`` (contiguous) where the caller brings it, ``residual`` itself to update it in place; any other
    overlap is refused."""
    return _dense("gemm_bias_act", a, b, None, None, bias, activation, False, scale, residual, out_dtype or a.dtype, out)


def gemm_act_and_mul(a: torch.Tensor, b: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "silu",
                     out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Both projections of a gated block, activation and product in one: ``out = act(a b[:I]^T + bias[:I]) * (a b[I:]^T + bias[I:])``
    with ``b`` [2I, K], the gate's rows first as in the experts' ``w1``; ``activation`` "silu" or "gelu".  Nothing of it is
    rounded before the result; the rest as in ``gemm_bias_act`` (tiles of 256 x 128 results)."""
    return _dense("gemm_act_and_mul", a, b, None, None, bias, activation, True, 1.0, None, out_dtype or a.dtype, out)


def gemm_w8a8_bias_act(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                       activation: Optional[str] = None, residual: Optional[torch.Tensor] = None, scale: float = 1.0,
                       out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``gemm_bias_act`` of int8 operands with a scale for each row of either, the per-channel form of the experts:
    ``out = scale * act((a b^T) * a_scale * b_scale + bias) + residual``, the sum exact in int32.

    ``a`` [..., K] with ``a_scale`` [...] or [..., 1] (``rms_norm_quant``, ``per_token_quant_int8``, ``fuse_silu_mul_quant``), ``b`` [N, K]
    row-major with ``b_scale`` [N] or [N, 1], scales fp32; K a multiple of 16 and at most 131056."""
    if a_scale is None or b_scale is None:
        raise RuntimeError("gemm_w8a8_bias_act: a_scale and b_scale must be tensors")
    return _dense("gemm_w8a8_bias_act", a, b, a_scale, b_scale, bias, activation, False, scale, residual, out_dtype, out)


def gemm_w8a8_act_and_mul(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor,
                          bias: Optional[torch.Tensor] = None, activation: str = "silu", out_dtype: torch.dtype = torch.bfloat16,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``gemm_act_and_mul`` of int8 operands with a scale for each row of either, as ``gemm_w8a8_bias_act`` takes them."""
    if a_scale is None or b_scale is None:
        raise RuntimeError("gemm_w8a8_act_and_mul: a_scale and b_scale must be tensors")
    return _dense("gemm_w8a8_act_and_mul", a, b, a_scale, b_scale, bias, activation, True, 1.0, None, out_dtype, out)


__all__ = ["moe_gemm_w8a8", "gemm_w8a8_fp8_block", "gemm_bias_act", "gemm_act_and_mul", "gemm_w8a8_bias_act", "gemm_w8a8_act_and_mul"]
