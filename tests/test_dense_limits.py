"""Sizes of the dense products: which have a kernel, which are refused, and that the queries say the same as the call.  Host only."""
import ctypes

import pytest

BF16, F16, I8 = 0, 1, 3
MOST_TILES = 1 << 22  # of a launch


@pytest.fixture(scope="module")
def lib():
    from lightop_amd import _lib

    return _lib.lib()


def _tile(lib, dtype, gated, M, N, K, workspace):
    a = [ctypes.c_int32() for _ in range(3)]
    return lib.lo_gemm_bias_act_tile_query(dtype, gated, M, N, K, workspace, *(ctypes.byref(v) for v in a)), tuple(v.value for v in a)


def _tiles(M, N, tm, tn, gated):
    width = tn // 2 if gated else tn
    return -(-M // tm) * -(-N // width)


@pytest.mark.parametrize("gated,M,N,K", [(0, 1 << 24, 4096, 64), (1, 11625891, 1635, 256), (1, 12000000, 1640, 16), (0, 8192, 1 << 23, 64), (0, 200000, 200003, 64),
                                         (1, 1 << 24, 8000, 512), (0, 1 << 24, 16384 - 256, 7168), (0, 17, 1 << 23, 128)])
def test_a_size_that_has_a_kernel_takes_it(lib, gated, M, N, K):
    """With short K the smaller tiles are the faster ones; more of them than a launch takes are none."""
    assert _tiles(M, N, 256, 256, gated) < MOST_TILES
    for dtype in (BF16, F16, I8):
        for workspace in (0, 1):
            rc, (tm, tn, parts) = _tile(lib, dtype, gated, M, N, K, workspace)
            assert rc == 0 and _tiles(M, N, tm, tn, gated) < MOST_TILES and (workspace or parts == 1)
        assert lib.lo_gemm_bias_act_workspace_bytes(dtype, gated, M, N, K) >= 0


@pytest.mark.parametrize("gated,M,N,K", [(0, 1 << 24, 1 << 23, 64), (0, 1 << 24, 16384, 64), (1, 1 << 24, 8192, 64), (0, 131072, 1 << 23, 7168), (1, 65536, 1 << 23, 16)])
def test_a_size_without_a_kernel_is_refused_everywhere(lib, gated, M, N, K):
    assert _tiles(M, N, 256, 256, gated) >= MOST_TILES
    p = 1 << 44  # stands for an aligned pointer, used by nobody
    for dtype in (BF16, I8):
        scale = p if dtype == I8 else None
        calls = (lambda: _tile(lib, dtype, gated, M, N, K, 1)[0], lambda: lib.lo_gemm_bias_act_workspace_bytes(dtype, gated, M, N, K),
                 lambda: lib.lo_gemm_bias_act(p, K, p, K, dtype, scale, scale, None, BF16, 0, gated, 1.0, None, 0, 1 << 50, BF16, M, N, K, None, 0, None))
        for call in calls:
            assert lib.lo_gemm_bias_act_tile_query(BF16, 0, 4, 32, 60, 1, None, None, None) == -1  # another error before it
            assert call() == -4 and b"2^22 tiles" in lib.lo_last_error()


def test_no_rows_and_no_columns_need_no_tiles(lib):
    assert _tile(lib, BF16, 0, 0, 1 << 23, 64, 1)[0] == 0 and _tile(lib, BF16, 1, 1 << 24, 0, 64, 1)[0] == 0
    assert lib.lo_gemm_bias_act_workspace_bytes(BF16, 0, 1 << 24, 0, 64) == 0 and lib.lo_gemm_bias_act_workspace_bytes(I8, 1, 0, 1 << 23, 64) == 0
