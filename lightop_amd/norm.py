"""RMS norm in front of a quantised layer: residual added, rows normed, 8 bits out.

The producer of what the layers take: int8 rows with one scale are the ``i_q`` / ``i_s`` of ``fused_experts_impl_int8``
(python/lightop/_lmslim_native/layers/fused_moe/int8.py:291-293, LMSLIM_USE_FUSED_RMS_QUANT), int8 rows with a scale for 128
values the ``A`` / ``A_scale`` of ``invoke_fused_moe_kernel_int8``, e4m3 rows those of ``gemmopt.gemm_w8a8_fp8_block``."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .op import _float_dtype, _on_device, _one_device, _rows16


class RmsNormQuant(NamedTuple):
    q: torch.Tensor                    # codes, the shape of x
    scale: torch.Tensor                # fp32, x.shape[:-1] + (1,) or (H // 128,)
    residual: Optional[torch.Tensor]   # x + residual in x's type
    normed: Optional[torch.Tensor]     # the normed rows in x's type


_FORMS = {(torch.int8, None): _lib.LO_Q_INT8_ROWS, (torch.int8, 128): _lib.LO_Q_INT8_GROUPS,
          (torch.float8_e4m3fn, 128): _lib.LO_Q_FP8_GROUPS}


def _strided_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as [rows, H] whose rows are contiguous and 16-byte aligned: a view where it can be."""
    t = t.reshape(-1, t.shape[-1])
    size = t.element_size()
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or (t.stride(0) >= t.shape[1]
                                                                            and t.stride(0) * size % 16 == 0)):
        return t
    return _rows16(t)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                   quant_dtype: torch.dtype = torch.int8, group_size: Optional[int] = None, return_normed: bool = False,
                   residual_out: Optional[torch.Tensor] = None) -> RmsNormQuant:
    """``z = x + residual``, ``y = z / sqrt(mean(z^2) + eps) * weight`` over the last dimension in fp32, and y's 8-bit
    codes and scales.

    ``quant_dtype=torch.int8, group_size=None``: one scale a row, the rule of ``per_token_quant_int8``;
    ``torch.int8, 128``: one for 128 values, the rule of ``per_token_group_quant_int8``;
    ``torch.float8_e4m3fn, 128``: the rule of ``per_token_group_quant_fp8``.  Codes are taken from the fp32 y.

    ``x`` bf16, fp16 or fp32 of any leading shape (rows may be strided), ``weight`` of its type or fp32.  The sum comes back
    in ``residual`` in x's type, in ``residual_out`` where the caller brings one (contiguous; ``residual`` itself updates it
    in place; any other overlap with rows that are read where they lie is refused), None without a residual; with
    ``return_normed`` the normed rows in x's type come back too."""
    form = _FORMS.get((quant_dtype, group_size))
    if form is None:
        raise RuntimeError("rms_norm_quant: built for int8 with group_size None or 128 and float8_e4m3fn with 128, "
                           f"got {quant_dtype} and {group_size}")
    made = (_lib._host or _lib.host()).rms_norm_quant(x, weight, residual, residual_out, eps, form, return_normed)
    if made is not None:  # None: not an ordinary call (csrc/host_binding.cpp); checked and converted below
        return RmsNormQuant(*made)
    _one_device(x, weight, residual, residual_out)
    H = x.shape[-1] if x.dim() else 0
    unit = 8 if group_size is None else group_size
    if H == 0 or H % unit:
        raise RuntimeError(f"rms_norm_quant: the last dimension of x must be a multiple of {unit}, got {tuple(x.shape)}")
    dtype = _float_dtype(x, "x")
    if weight.shape != (H,) or weight.dtype not in (x.dtype, torch.float32):
        raise RuntimeError("rms_norm_quant: weight must be [hidden], of x's type or float32")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise RuntimeError("rms_norm_quant: residual must have the shape and type of x")
    if residual_out is not None and (residual is None or residual_out.shape != x.shape or residual_out.dtype != x.dtype
                                     or not residual_out.is_contiguous()):
        raise RuntimeError("rms_norm_quant: residual_out goes with a residual, contiguous and of x's shape and type")
    q = torch.empty(x.shape, dtype=quant_dtype, device=x.device)
    scale = torch.empty(x.shape[:-1] + (1 if group_size is None else H // group_size,), dtype=torch.float32, device=x.device)
    total = None
    if residual is not None:
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual_out is None else residual_out
    normed = torch.empty(x.shape, dtype=x.dtype, device=x.device) if return_normed else None
    if x.numel() == 0:
        return RmsNormQuant(q, scale, total, normed)
    rows, w = _strided_rows(x), _rows16(weight)
    res = None if residual is None else _strided_rows(residual)
    target = total  # (contiguous rows that begin off 16 bytes take a copy, as inputs do)
    if total is not None and total.data_ptr() % 16:
        target = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with _on_device(x):
        _lib.check(_lib.lib().lo_rms_norm_quant(
            _lib.ptr(rows), dtype, rows.stride(0), _lib.ptr(res), 0 if res is None else res.stride(0), _lib.ptr(w),
            _float_dtype(w, "weight"), rows.shape[0], H, float(eps), form, _lib.ptr(target), _lib.ptr(normed), _lib.ptr(q),
            _lib.ptr(scale), _lib.stream_of(x)))
        if target is not total:
            total.detach().copy_(target)
    return RmsNormQuant(q, scale, total, normed)


__all__ = ["RmsNormQuant", "rms_norm_quant"]
