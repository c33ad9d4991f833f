"""What the dense blocks' operators refuse, before any GPU call: through the C entry points, and through Python on CPU tensors."""
import ctypes

import pytest
import torch

import dense_ref as ref


@pytest.fixture(scope="module")
def lib():
    from lightop_amd import _lib

    return _lib.lib()


P = 1 << 40  # stands for an aligned pointer; nothing below gets as far as using it
FAR = P + (1 << 36)
BF16, F16, F32, I8 = 0, 1, 2, 3


def _gemm(lib, **k):
    a = dict(a=P, sa=64, b=P + (1 << 30), sb=64, dt=BF16, xa=0, xb=0, bias=0, bt=BF16, act=-1, gated=0, scale=1.0, r=0, rs=0, c=FAR, out=BF16, M=4,
             N=32, K=64, ws=0, n=0)
    if k.get("dt") == I8:
        a.update(xa=P + (1 << 31), xb=P + (1 << 32))
    a.update(k)
    return lib.lo_gemm_bias_act(a["a"], a["sa"], a["b"], a["sb"], a["dt"], a["xa"], a["xb"], a["bias"], a["bt"], a["act"], a["gated"], a["scale"],
                                a["r"], a["rs"], a["c"], a["out"], a["M"], a["N"], a["K"], a["ws"], a["n"], None)


@pytest.mark.parametrize("bad", [
    dict(dt=F32), dict(dt=4), dict(M=-1), dict(N=-1), dict(K=0), dict(K=60), dict(dt=I8, K=56), dict(dt=I8, K=131072, sa=131072, sb=131072),
    dict(K=1 << 22), dict(M=1 << 25), dict(N=1 << 24), dict(out=I8), dict(act=2), dict(act=-2), dict(bias=P, bt=F16), dict(a=0), dict(b=0), dict(c=0),
    dict(dt=I8, xa=0), dict(dt=I8, xb=0), dict(xa=P, xb=P), dict(sa=56), dict(sb=56), dict(r=P, rs=31), dict(sa=68), dict(sb=68), dict(sa=1 << 22),
    dict(a=P + 8), dict(b=P + 2), dict(c=FAR + 1), dict(out=F32, c=FAR + 2), dict(r=P + 1, rs=32), dict(bias=P + 1), dict(bias=P + 2, bt=F32),
    dict(dt=I8, xa=P + 2), dict(ws=P + 8, n=64), dict(ws=P, n=-1), dict(c=P + 64), dict(b=FAR - 64), dict(dt=I8, xa=FAR), dict(bias=FAR + 16, bt=F32),
    dict(r=FAR + 64, rs=32), dict(r=FAR, rs=64), dict(gated=1, b=FAR - 32 * 128 - 64)], ids=str)
def test_gemm_refuses(lib, bad):
    assert _gemm(lib, **bad) < 0
    assert b"gemm_bias_act" in lib.lo_last_error()


@pytest.mark.parametrize("bad", [dict(dtype=F32), dict(K=0), dict(K=60), dict(M=-1), dict(N=-1), dict(N=1 << 24), dict(M=1 << 25), dict(K=1 << 22),
                                 dict(dtype=I8, K=131072)], ids=str)
def test_the_workspace_query_refuses_what_the_call_refuses(lib, bad):
    a = dict(dtype=BF16, gated=0, M=4, N=32, K=64)
    a.update(bad)
    assert _gemm(lib, dt=7) < 0  # another error before it
    assert lib.lo_gemm_bias_act_workspace_bytes(a["dtype"], a["gated"], a["M"], a["N"], a["K"]) < 0
    assert b"gemm_bias_act" in lib.lo_last_error()


def _norm(lib, **k):
    a = dict(x=P, dt=BF16, xs=256, r=P + (1 << 20), rs=256, post=0, pt=BF16, gate=0, gt=BF16, gs=0, rows=1, chan=0, sig=0, w=P + (1 << 22), wt=BF16,
             scale=1.0, rscale=1.0, M=2, H=256, eps=1e-6, form=0, z=FAR, y=0, q=P, s=P)
    a.update(k)
    return lib.lo_rms_norm_block(a["x"], a["dt"], a["xs"], a["r"], a["rs"], a["post"], a["pt"], a["gate"], a["gt"], a["gs"], a["rows"], a["chan"],
                                 a["sig"], a["w"], a["wt"], a["scale"], a["rscale"], a["M"], a["H"], a["eps"], a["form"], a["z"], a["y"], a["q"], a["s"],
                                 None)


@pytest.mark.parametrize("bad", [
    dict(M=-1), dict(M=1 << 31), dict(dt=3), dict(wt=F16), dict(post=P, pt=F16), dict(gate=P, gt=F16), dict(form=3), dict(form=-2), dict(H=0), dict(H=260),
    dict(form=1, H=264), dict(form=2, H=8), dict(H=65544), dict(eps=-1.0), dict(eps=float("nan")), dict(w=0), dict(w=0, form=-1, y=P),
    dict(gate=P, rows=0), dict(gate=P, gs=-256), dict(x=0), dict(r=0), dict(z=0), dict(q=0), dict(s=0), dict(form=-1), dict(xs=128), dict(rs=0),
    dict(xs=260), dict(rs=260), dict(gate=P, chan=1, gs=260), dict(x=P + 2), dict(r=P + 4), dict(w=P + 8), dict(post=P + 8), dict(z=FAR + 4), dict(y=P + 4),
    dict(q=P + 4), dict(s=P + 2), dict(gate=P + 2, chan=1), dict(gate=P + 1), dict(gate=P + 2, gt=F32)], ids=str)
def test_norm_refuses(lib, bad):
    assert _norm(lib, **bad) < 0
    assert b"rms_norm_block" in lib.lo_last_error()


@pytest.mark.parametrize("bad", [dict(z=P + 512), dict(z=P - 512), dict(z=P + (1 << 20) + 16), dict(z=P, xs=512), dict(z=P + (1 << 20), rs=512),
                                 dict(w=FAR + 16), dict(post=FAR - 16), dict(gate=FAR, chan=1, gs=256), dict(gate=FAR + 512, gs=1),
                                 dict(gate=FAR - 2, gs=1), dict(M=1, z=P + 16)], ids=str)
def test_norm_refuses_a_sum_over_an_input(lib, bad):
    assert _norm(lib, **bad) < 0
    assert b"overlaps" in lib.lo_last_error()


def test_no_rows_is_no_error(lib):
    assert _norm(lib, M=0, x=0, r=0, z=0, q=0, s=0) == 0
    assert _gemm(lib, M=0, a=0, c=0) == 0 and _gemm(lib, N=0, b=0, c=0) == 0
    assert lib.lo_gemm_bias_act_workspace_bytes(BF16, 0, 0, 32, 64) == 0 and lib.lo_gemm_bias_act_workspace_bytes(I8, 1, 100, 0, 64) == 0


def test_python_needs_the_gpu():
    from lightop_amd import gemmopt
    from lightop_amd.norm import rms_norm_block

    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    i, s = torch.zeros(2, 256, dtype=torch.int8), torch.zeros(2)
    for call in (lambda: rms_norm_block(x, x, x[0]), lambda: gemmopt.gemm_bias_act(x, x), lambda: gemmopt.gemm_act_and_mul(x, x),
                 lambda: gemmopt.gemm_w8a8_bias_act(i, i, s, s), lambda: gemmopt.gemm_w8a8_act_and_mul(i, i, s, s)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(RuntimeError, match="group_size"):
        rms_norm_block(x, x, x[0], quant_dtype=torch.float8_e4m3fn)
    with pytest.raises(ValueError):
        gemmopt.gemm_bias_act(x, x, activation="relu")


def test_names_are_reachable():
    import lightop
    import lightop.gemmopt
    import lightop.norm
    import lightop_amd

    assert lightop.norm.rms_norm_block is lightop_amd.norm.rms_norm_block
    for name in ("gemm_bias_act", "gemm_act_and_mul", "gemm_w8a8_bias_act", "gemm_w8a8_act_and_mul"):
        assert getattr(lightop.gemmopt, name) is getattr(lightop_amd.gemmopt, name) and name in lightop_amd.gemmopt.__all__


def _tile(lib, dtype, gated, M, N, K, workspace):
    a = [ctypes.c_int32() for _ in range(3)]
    assert lib.lo_gemm_bias_act_tile_query(dtype, gated, M, N, K, workspace, *(ctypes.byref(v) for v in a)) == 0
    return tuple(v.value for v in a)


@pytest.mark.parametrize("tile,size", ref.TILE_SIZES, ids=str)
def test_tile_of_the_sizes_that_the_gpu_tests_take(lib, tile, size):
    M, N, K = size
    tm, tn, split, gated = tile
    for dtype, k in ((BF16, K), (F16, K), (I8, 2 * K)):
        assert _tile(lib, dtype, gated, M, N, k, 1)[:2] == (tm, tn) and (_tile(lib, dtype, gated, M, N, k, 1)[2] > 1) == split
        assert (lib.lo_gemm_bias_act_workspace_bytes(dtype, gated, M, N, k) > 0) == split
        assert _tile(lib, dtype, gated, M, N, k, 0)[2] == 1


def test_every_tile_has_sizes(lib):
    """Over many sizes no call takes a tile, whole or in parts, that the list above leaves out, but for 128 x 256 in parts and the kernel of few tokens."""
    seen = set()
    for M in (9, 17, 33, 65, 100, 200, 400, 800, 1600, 3200, 8000):
        for N in (16, 40, 130, 300, 577, 1000, 2000, 4100, 8000):
            for K in (16, 200, 504, 1000, 2000, 4000, 8000):
                for gated in (0, 1):
                    tm, tn, parts = _tile(lib, BF16, gated, M, N, K, 1)
                    seen.add((tm, tn, parts > 1, bool(gated)))
    assert seen <= set(ref.TILES) | {(128, 256, True, False), (128, 256, True, True), (16, 16, False, False), (16, 16, False, True)}
    assert all(_tile(lib, BF16, gated, M, N, K, 1) == (16, 16, 1) for M, N, K, gated in ref.FEW)
    assert all(_tile(lib, I8 if M > 8 else BF16, 0, M, 2048, 256, 1) == (16, 16, 1) for M in (1, 8, 16))


def test_tile_query_refuses(lib):
    v = ctypes.byref(ctypes.c_int32())
    assert lib.lo_gemm_bias_act_tile_query(BF16, 0, 4, 32, 60, 1, v, v, v) < 0 and lib.lo_gemm_bias_act_tile_query(BF16, 0, 4, 32, 64, 1, v, None, v) < 0
    assert b"gemm_bias_act" in lib.lo_last_error()
    assert lib.lo_gemm_bias_act_tile_query(BF16, 0, 0, 0, 64, 1, v, v, v) == 0
