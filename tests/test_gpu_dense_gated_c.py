"""Gated dense products with a scale and a residual, which the C entry point takes (the Python ones have no use for them): scale * act(gate) * up + residual."""
import pytest
import torch

import dense_parts as parts
import dense_ref as ref

pytestmark = pytest.mark.gpu

FEW = [s[:3] for s in ref.FEW if s[3]]
TILES = [size for tile, sizes in ref.TILES.items() if tile[3] for size in sizes]


def _call(kind, ops, bias, name, scale, r, out, N):
    from lightop_amd import _lib

    a, b, sa, sb = ops
    (M, K), lib, kinds = a.shape, _lib.lib(), {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
    need = lib.lo_gemm_bias_act_workspace_bytes(parts.CODES[kind], 1, M, N, K)
    room = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    _lib.check(lib.lo_gemm_bias_act(_lib.ptr(a), K, _lib.ptr(b), K, parts.CODES[kind], _lib.ptr(sa), _lib.ptr(sb), _lib.ptr(bias), kinds[bias.dtype],
                                    {None: -1, "silu": 0, "gelu": 1}[name], 1, scale, _lib.ptr(r), r.stride(0), _lib.ptr(out), kinds[out.dtype], M, N, K,
                                    _lib.ptr(room), need, _lib.stream_of(a)))
    return out


@pytest.mark.parametrize("size", FEW + TILES, ids=str)
def test_scale_and_residual(size):
    M, N, K = size
    for kind, dtype, name, k in ((torch.bfloat16, torch.bfloat16, "silu", K), (torch.float16, torch.float32, None, K), (torch.int8, torch.float16, "gelu", 2 * K)):
        print("[case] gated", kind, M, N, k, flush=True)
        g = torch.Generator(device="cuda").manual_seed(M + N + k)
        ops = ref.operands(kind, M, 2 * N, k, g)
        bias = torch.randn(2 * N, generator=g, device="cuda")
        r = torch.randn(M, N, generator=g, device="cuda").to(dtype)
        want = ref.dense(*ops, bias, name, True, r, -0.75)
        got = _call(kind, ops, bias, name, -0.75, r, torch.empty_like(r), N)
        ref.check(got, want)
        for left, more in ((8, 24), (5, 27)):
            wide = torch.full((M, N + more), float("nan"), dtype=dtype, device="cuda")
            wide[:, left:left + N] = r
            assert torch.equal(_call(kind, ops, bias, name, -0.75, wide[:, left:left + N], torch.empty_like(r), N), got)
        place = r.clone()
        assert torch.equal(_call(kind, ops, bias, name, -0.75, place, place, N), got)
