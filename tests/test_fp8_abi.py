"""What the 8-bit operators refuse, before any GPU call: through the C entry points, and through Python on CPU tensors."""
import ctypes

import pytest
import torch

import fp8_ref as ref


@pytest.fixture(scope="module")
def lib():
    from lightop_amd import _lib

    return _lib.lib()


P = 4096  # stands for an aligned pointer; nothing below gets as far as using it


def _norm(lib, **k):
    a = dict(x=P, dtype=0, xs=256, r=P, rs=256, w=P, wt=0, M=2, H=256, eps=1e-6, form=0, z=P, y=0, q=P, s=P)
    a.update(k)
    return lib.lo_rms_norm_quant(a["x"], a["dtype"], a["xs"], a["r"], a["rs"], a["w"], a["wt"], a["M"], a["H"], a["eps"], a["form"], a["z"],
                                 a["y"], a["q"], a["s"], None)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(wt=1), dict(form=3), dict(form=-1), dict(H=0), dict(H=260), dict(form=1, H=264),
                                 dict(form=2, H=8), dict(H=65544), dict(eps=-1.0), dict(eps=float("nan")), dict(x=0), dict(w=0), dict(q=0),
                                 dict(s=0), dict(z=0), dict(M=-1), dict(xs=128), dict(rs=0), dict(xs=260), dict(x=P + 2), dict(w=P + 8),
                                 dict(q=P + 4), dict(s=P + 2), dict(z=P + 4), dict(y=P + 4), dict(r=P + 4)], ids=str)
def test_norm_refuses(lib, bad):
    assert _norm(lib, **bad) < 0
    assert b"rms_norm_quant" in lib.lo_last_error()


def test_no_rows_is_no_error(lib):
    assert _norm(lib, M=0, x=0, w=0, q=0, s=0, z=0) == 0
    assert lib.lo_per_token_group_quant_fp8(None, 0, 0, 128, 1e-10, None, None, None) == 0
    assert lib.lo_act_mul_group_quant_fp8(None, 0, 0, 0, 128, None, None, None) == 0
    assert lib.lo_gemm_w8a8_fp8_block(None, None, None, None, None, 0, 0, 128, 128, None, 0, None) == 0
    assert lib.lo_gemm_w8a8_fp8_block(None, None, None, None, None, 0, 128, 0, 128, None, 0, None) == 0
    assert _experts(lib, M=0, x=0, out=0, ws=0) == 0


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(rows=-1), dict(cols=0), dict(cols=192), dict(x=0), dict(q=0), dict(s=0), dict(x=P + 8),
                                 dict(q=P + 4), dict(s=P + 1), dict(eps=0.0), dict(eps=1e-31), dict(eps=float("inf")), dict(eps=float("nan"))],
                         ids=str)
def test_group_quant_refuses(lib, bad):
    a = dict(x=P, dtype=0, rows=1, cols=128, eps=1e-10, q=P, s=P)
    a.update(bad)
    assert lib.lo_per_token_group_quant_fp8(a["x"], a["dtype"], a["rows"], a["cols"], a["eps"], a["q"], a["s"], None) < 0
    if "eps" not in bad:
        assert lib.lo_act_mul_group_quant_fp8(a["x"], a["dtype"], 0, a["rows"], a["cols"], a["q"], a["s"], None) < 0
    assert b"group_quant_fp8" in lib.lo_last_error()


def test_act_refuses_unknown_activation(lib):
    assert lib.lo_act_mul_group_quant_fp8(P, 0, 2, 1, 128, P, P, None) < 0


@pytest.mark.parametrize("bad", [dict(M=-1), dict(N=-1), dict(K=0), dict(K=64), dict(K=1 << 23), dict(M=1 << 25), dict(N=1 << 25),
                                 dict(dt=3), dict(a=0), dict(b=0), dict(sa=0), dict(sb=0), dict(c=0), dict(a=P + 8), dict(b=P + 1),
                                 dict(sa=P + 2), dict(c=P + 1), dict(ws=P + 8, n=64), dict(ws=P, n=-1)], ids=str)
def test_gemm_refuses(lib, bad):
    a = dict(a=P, sa=P, b=P, sb=P, c=P, dt=0, M=1, N=16, K=128, ws=0, n=0)
    a.update(bad)
    assert lib.lo_gemm_w8a8_fp8_block(a["a"], a["sa"], a["b"], a["sb"], a["c"], a["dt"], a["M"], a["N"], a["K"], a["ws"], a["n"],
                                      None) < 0
    assert b"gemm_w8a8_fp8_block" in lib.lo_last_error()


def _experts(lib, **k):
    a = dict(x=P, dt=0, M=2, H=256, I=128, E=4, Eg=4, top_k=2, w1=P, s1=P, w2=P, s2=P, tw=P, ids=P, it=0, map=0, act=0, sh=0, out=P, ws=P,
             n=1 << 20)
    a.update(k)
    return lib.lo_fused_experts_fp8(a["x"], a["dt"], a["M"], a["H"], a["I"], a["E"], a["Eg"], a["top_k"], a["w1"], a["s1"], a["w2"], a["s2"],
                                    a["tw"], a["ids"], a["it"], a["map"], a["act"], 1.0, a["sh"], a["out"], a["ws"], a["n"], None)


@pytest.mark.parametrize("bad", [dict(dt=2), dict(it=2), dict(act=2), dict(M=-1), dict(H=64), dict(H=320), dict(I=64), dict(E=0), dict(Eg=3),
                                 dict(Eg=8), dict(top_k=0), dict(M=65), dict(M=64, top_k=17), dict(M=1, top_k=65), dict(x=0), dict(w1=0), dict(w2=0), dict(s1=0),
                                 dict(s2=0), dict(tw=0), dict(ids=0), dict(out=0), dict(ws=0), dict(n=100), dict(x=P + 8), dict(ws=P + 4),
                                 dict(w2=P + 4), dict(E=4096, Eg=4096), dict(H=1 << 21)], ids=str)
def test_experts_refuses(lib, bad):
    assert _experts(lib, **bad) < 0
    assert b"fused_experts_fp8" in lib.lo_last_error()


def test_gemm_workspace(lib):
    n = lib.lo_gemm_w8a8_fp8_block_workspace_bytes
    assert n(1, 4096, 7168, 0) == 0 and n(8192, 4096, 7168, 0) == 0  # no parts
    assert n(333, 576, 7168, 0) > 0 and n(333, 576, 7168, 0) % (333 * 576 * 4) == 0
    assert n(333, 575, 7168, 0) % (333 * 576 * 4) == 0               # rows of a part begin on 16 bytes
    assert n(-1, 16, 128, 0) < 0 and n(1, 16, 100, 0) < 0 and n(100, 0, 128, 0) == 0


def test_experts_workspace(lib):
    n = lib.lo_fused_experts_fp8_workspace_bytes
    assert n(1, 8, 2048, 768) == 8 * 768 * 4
    assert n(64, 8, 7168, 2048) == 512 * 2048 * 4 + 64 * 7168 * (1 + 4 / 128) + 512 * 2048 * (1 + 4 / 128)
    assert n(-1, 8, 2048, 768) < 0 and n(1, 0, 2048, 768) < 0 and n(1, 1, 256, 64) < 0 and n(1, 1, 64, 256) < 0


def test_python_needs_the_gpu():
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block
    from lightop_amd.moe import act_and_mul_group_quant_fp8, fused_experts_decode_fp8
    from lightop_amd.norm import rms_norm_quant
    from lightop_amd.quant import per_token_group_quant_fp8

    x, f8 = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(256, 256).to(torch.float8_e4m3fn)
    s = torch.zeros(2, 2)
    for call in (lambda: rms_norm_quant(x, x[0]), lambda: per_token_group_quant_fp8(x, 128), lambda: act_and_mul_group_quant_fp8(x),
                 lambda: gemm_w8a8_fp8_block(f8[:2], f8, s, s),
                 lambda: fused_experts_decode_fp8(x, f8[None], f8[None, :, :128], s, s.int(), s[None], s[None, :, :1])):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(RuntimeError, match="group_size"):
        rms_norm_quant(x, x[0], quant_dtype=torch.float8_e4m3fn)
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        per_token_group_quant_fp8(x, 128, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="128"):
        per_token_group_quant_fp8(x, 64)
    with pytest.raises(ValueError):
        act_and_mul_group_quant_fp8(x, "relu")


def test_names_are_reachable():
    import lightop
    import lightop.norm
    import lightop_amd

    assert lightop.norm.rms_norm_quant is lightop_amd.norm.rms_norm_quant is lightop.rms_norm_quant
    assert lightop.moe.fused_experts_decode_fp8 is lightop_amd.moe.fused_experts_decode_fp8
    assert lightop.gemmopt.gemm_w8a8_fp8_block and lightop.quant.per_token_group_quant_fp8


@pytest.mark.parametrize("bad", [dict(z=P + 512), dict(z=P - 512), dict(x=P + 512, r=P + 1024 * 1024, z=P), dict(x=P + 1024 * 1024, r=P + 16, z=P),
                                 dict(xs=512), dict(rs=512), dict(M=1, z=P + 16), dict(dtype=2, wt=2, z=P + 1024)], ids=str)
def test_norm_refuses_a_sum_over_other_rows(lib, bad):
    assert _norm(lib, **bad) < 0
    assert b"overlaps" in lib.lo_last_error()


@pytest.mark.parametrize("M,top_k,H,I", [(65, 1, 256, 128), (8192, 8, 7168, 2048), (2 ** 62, 64, 256, 128), (64, 17, 256, 128), (1, 65, 256, 128),
                                         (1, 0, 256, 128), (1, 1, 1 << 21, 128), (1, 1, 256, 1 << 21), (1, 1, 320, 128), (1, 1, 256, 192)])
def test_experts_workspace_refuses_what_the_call_refuses(lib, M, top_k, H, I):
    """Whoever sizes the workspace first meets the refusal before taking memory for it."""
    assert lib.lo_gemm_w8a8_fp8_block(0, 0, 0, 0, 0, 0, -1, 1, 128, 0, 0, None) < 0  # another operator's error before it
    assert lib.lo_fused_experts_fp8_workspace_bytes(M, top_k, H, I) < 0
    assert b"fused_experts_fp8" in lib.lo_last_error()


@pytest.mark.parametrize("M,N,K,dtype", [((1 << 24) + 1, 16, 128, 0), (2 ** 62, 2 ** 62, 128, 0), (100, (1 << 24) + 1, 128, 0), (100, 16, 1 << 23, 0),
                                         (100, 16, 64, 0), (-1, 16, 128, 0), (100, 16, 128, 3)])
def test_gemm_workspace_refuses_what_the_call_refuses(lib, M, N, K, dtype):
    assert lib.lo_per_token_group_quant_fp8(None, 7, 0, 128, 1e-10, None, None, None) < 0  # another operator's error before it
    assert lib.lo_gemm_w8a8_fp8_block_workspace_bytes(M, N, K, dtype) < 0
    assert b"gemm_w8a8_fp8_block" in lib.lo_last_error()


@pytest.mark.parametrize("out,sh", [(P + 2, P), (P, P + 2), (P + 1022, P), (P, P + 512)])
def test_experts_refuse_shared_rows_under_other_outputs(lib, out, sh):
    """Two rows of 256: an output stored over a shared value that another one still adds."""
    assert _experts(lib, out=out, sh=sh) < 0
    assert b"overlaps" in lib.lo_last_error()


def _tile(lib, M, N, K, dtype=0, workspace=1):
    out = [ctypes.c_int32(-7) for _ in range(3)]
    rc = lib.lo_gemm_w8a8_fp8_block_tile_query(M, N, K, dtype, workspace, *(ctypes.byref(v) for v in out))
    return rc if rc else tuple(v.value for v in out)


def test_tiles_of_the_product(lib):
    """The sizes that the GPU tests run by tile take that tile, the list has every tile that there is, and the workspace holds the parts."""
    seen = {(16, 16, False)}
    assert _tile(lib, 1, 4096, 7168) == _tile(lib, 16, 30, 128) == (16, 16, 1)
    for (tm, tn, parts), (M, N, K) in ref.TILE_SIZES:
        for dtype in (0, 1, 2):
            m, n, p = _tile(lib, M, N, K, dtype)
            assert (dtype == 2 and tm * tn > 128 * 128) or ((m, n, p > 1) == (tm, tn, parts)), (M, N, K, dtype)
            seen.add((m, n, p > 1))
            need = lib.lo_gemm_w8a8_fp8_block_workspace_bytes(M, N, K, dtype)
            assert need == (p * M * -(-N // 4) * 16 if p > 1 else 0)
            assert _tile(lib, M, N, K, dtype, 0)[2] == 1
    for M in (17, 20, 33, 64, 65, 100, 128, 200, 300, 500, 800, 1400, 3000, 8192):
        for N in (1, 24, 576, 1000, 2048, 4097, 7168, 16384):
            for K in (128, 512, 1152, 2048, 7168, 16384):
                for dtype in (0, 2):
                    m, n, p = _tile(lib, M, N, K, dtype)
                    assert (m, n, p > 1) in seen
    for bad in ((-1, 1, 128), (1, 1, 64), (1, (1 << 24) + 1, 128), (1, 1, 1 << 23), (20, 20, 128, 3)):
        assert _tile(lib, *bad) < 0 and b"gemm_w8a8_fp8_block" in lib.lo_last_error()
    assert lib.lo_gemm_w8a8_fp8_block_tile_query(1, 1, 128, 0, 1, None, None, None) < 0
