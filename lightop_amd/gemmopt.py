"""Grouped-GEMM stage of the per-channel W8A8 MoE, and the dense e4m3 product with block scales (reference: lightop.gemmopt.moe_gemm_w8a8,
python/lightop/gemmopt.py:437-457; native side csrc/moe_gemm/w8a8/moe_w8a8.cu:2389-2536)."""
from __future__ import annotations

from typing import Any, Dict, Optional

import torch

from . import _lib
from .op import _act_dtype, _on_device, _one_device, _require_cuda, _rows16


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


__all__ = ["moe_gemm_w8a8", "gemm_w8a8_fp8_block"]
