"""RMS norm in front of a quantised layer: residual added, rows normed, 8 bits out; and the norms on both sides of a block.

The producer of what the layers take: int8 rows with one scale are the ``i_q`` / ``i_s`` of ``fused_experts_impl_int8``
(python/lightop/_lmslim_native/layers/fused_moe/int8.py:291-293, LMSLIM_USE_FUSED_RMS_QUANT), int8 rows with a scale for 128
values the ``A`` / ``A_scale`` of ``invoke_fused_moe_kernel_int8``, e4m3 rows those of ``gemmopt.gemm_w8a8_fp8_block``."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .op import _float_dtype, _on_device, _one_device, _rows16, _strided_rows


class RmsNormQuant(NamedTuple):
    q: torch.Tensor                    # codes, the shape of x
    scale: torch.Tensor                # fp32, x.shape[:-1] + (1,) or (H // 128,)
    residual: Optional[torch.Tensor]   # x + residual in x's type
    normed: Optional[torch.Tensor]     # the normed rows in x's type


_FORMS = {(torch.int8, None): _lib.LO_Q_INT8_ROWS, (torch.int8, 128): _lib.LO_Q_INT8_GROUPS,
          (torch.float8_e4m3fn, 128): _lib.LO_Q_FP8_GROUPS}


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


class RmsNormBlock(NamedTuple):
    residual: torch.Tensor             # the sum, in x's type
    normed: Optional[torch.Tensor]     # the normed sum in x's type
    q: Optional[torch.Tensor]          # its codes, the shape of x
    scale: Optional[torch.Tensor]      # fp32, x.shape[:-1] + (1,) or (H // 128,)


_GATES = {None: 0, "sigmoid": 1}


def _gate_rows(gate: torch.Tensor, x: torch.Tensor):
    """``gate`` as rows that ``rms_norm_block`` finds by a division: (tensor, row stride, rows of x that share a row)."""
    width = gate.shape[-1]
    lead = gate.expand(x.shape[:-1] + (width,))
    aligned = width == 1 or (gate.stride(-1) == 1 and gate.data_ptr() % 16 == 0)
    # leading dimensions from the last: the ones that are broadcast share a row, the others have to follow each other
    shared, stride, span = 1, 0, 0
    for n, st in zip(reversed(lead.shape[:-1]), reversed(lead.stride()[:-1])):
        if n == 1:
            continue
        if stride == 0 and st == 0:
            shared *= n
        elif stride == 0:
            stride, span = st, n * st
        elif st == span:
            span *= n
        else:
            aligned = False
    if aligned and (width == 1 or stride * gate.element_size() % 16 == 0):
        return gate, stride, shared
    return _rows16(lead), width, 1


def rms_norm_block(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
                   post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                   gate_activation: Optional[str] = None, scale: float = 1.0, residual_scale: float = 1.0, eps: float = 1e-6,
                   quant_dtype: Optional[torch.dtype] = None, group_size: Optional[int] = None, return_normed: bool = False,
                   residual_out: Optional[torch.Tensor] = None) -> RmsNormBlock:
    """What lies between two blocks: the norm behind the first, its gate and the residual, the norm in front of the second; over
    the last dimension, in fp32, in one pass:
    ``h = x / sqrt(mean(x^2) + eps) * post_weight`` (``h = x`` without ``post_weight``),
    ``z = residual_scale * residual + scale * act(gate) * h`` (``act``: none, or ``gate_activation="sigmoid"``),
    ``y = z / sqrt(mean(z^2) + eps) * weight``, from the fp32 z.

    ``x`` and ``residual`` bf16, fp16 or fp32 of one shape (rows may be strided, fewer than 2^31), the last dimension a multiple of 8 up to 65536; ``weight``,
    ``post_weight`` [H] and ``gate`` of their type or fp32.  ``gate`` is broadcast to x: [..., 1] a value for a token, [H] or
    [batch, 1, H] one for a channel, x's shape one for each.

    ``z`` comes back in ``residual``, in ``residual_out`` where the caller brings one (contiguous; ``residual`` or ``x`` itself is
    updated in place, any other overlap refused).  ``quant_dtype`` and ``group_size`` as in ``rms_norm_quant`` give y's codes in ``q`` and
    ``scale`` and, with ``return_normed``, y in x's type; without ``quant_dtype`` y comes in ``normed``.  Without ``weight`` the
    call ends with z."""
    form = _lib.LO_Q_NONE if quant_dtype is None and group_size is None else _FORMS.get((quant_dtype, group_size))
    if form is None:
        raise RuntimeError("rms_norm_block: built for quant_dtype None, int8 with group_size None or 128 and float8_e4m3fn with 128, "
                           f"got {quant_dtype} and {group_size}")
    if gate_activation not in _GATES:
        raise ValueError(f"rms_norm_block: unsupported gate_activation {gate_activation!r}")
    if weight is None and (form != _lib.LO_Q_NONE or return_normed):
        raise RuntimeError("rms_norm_block: normed rows and codes need the weight of the norm")
    made = (_lib._host or _lib.host()).rms_norm_block(x, residual, weight, post_weight, gate, residual_out, _GATES[gate_activation], scale,
                                                      residual_scale, eps, form, return_normed)
    if made is not None:  # None: not an ordinary call (csrc/host_binding.cpp); checked and converted below
        return RmsNormBlock(*(made if residual_out is None else (residual_out, *made[1:])))
    _one_device(x, residual, weight, post_weight, gate, residual_out)
    H = x.shape[-1] if x.dim() else 0
    unit = 8 if group_size is None else group_size
    if H == 0 or H % unit:
        raise RuntimeError(f"rms_norm_block: the last dimension of x must be a multiple of {unit}, got {tuple(x.shape)}")
    dtype = _float_dtype(x, "x")
    for w in (weight, post_weight):
        if w is not None and (w.shape != (H,) or w.dtype not in (x.dtype, torch.float32)):
            raise RuntimeError("rms_norm_block: weight and post_weight must be [hidden], of x's type or float32")
    if residual.shape != x.shape or residual.dtype != x.dtype:
        raise RuntimeError("rms_norm_block: residual must have the shape and type of x")
    if gate is not None:
        lead = gate.shape[:-1]
        if gate.dim() == 0 or gate.dim() > x.dim() or gate.shape[-1] not in (1, H) or gate.dtype not in (x.dtype, torch.float32) \
                or any(n not in (1, m) for n, m in zip(reversed(lead), reversed(x.shape[:-1]))):
            raise RuntimeError(f"rms_norm_block: gate must broadcast to x, of x's type or float32, got {tuple(gate.shape)} {gate.dtype}")
    if residual_out is not None and (residual_out.shape != x.shape or residual_out.dtype != x.dtype or not residual_out.is_contiguous()):
        raise RuntimeError("rms_norm_block: residual_out must be contiguous and of x's shape and type")
    total = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual_out is None else residual_out
    q = codes = None
    if form != _lib.LO_Q_NONE:
        q = torch.empty(x.shape, dtype=quant_dtype, device=x.device)
        codes = torch.empty(x.shape[:-1] + (1 if group_size is None else H // group_size,), dtype=torch.float32, device=x.device)
    normed = None
    if weight is not None and (return_normed or form == _lib.LO_Q_NONE):
        normed = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return RmsNormBlock(total, normed, q, codes)
    rows, res = _strided_rows(x), _strided_rows(residual)
    w, post = (None if t is None else _rows16(t) for t in (weight, post_weight))
    g, gate_stride, shared = (None, 0, 1) if gate is None else _gate_rows(gate, x)
    target = total  # (contiguous rows that begin off 16 bytes take a copy, as inputs do)
    if total.data_ptr() % 16:
        target = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    code = lambda t: dtype if t is None else _float_dtype(t, "weight")
    with _on_device(x):
        _lib.check(_lib.lib().lo_rms_norm_block(
            _lib.ptr(rows), dtype, rows.stride(0), _lib.ptr(res), res.stride(0), _lib.ptr(post), code(post), _lib.ptr(g), code(g),
            gate_stride, shared, int(g is not None and g.shape[-1] != 1), _GATES[gate_activation], _lib.ptr(w), code(w), float(scale),
            float(residual_scale), rows.shape[0], H, float(eps), form, _lib.ptr(target), _lib.ptr(normed), _lib.ptr(q), _lib.ptr(codes),
            _lib.stream_of(x)))
        if target is not total:
            total.detach().copy_(target)
    return RmsNormBlock(total, normed, q, codes)


__all__ = ["RmsNormQuant", "RmsNormBlock", "rms_norm_quant", "rms_norm_block"]
