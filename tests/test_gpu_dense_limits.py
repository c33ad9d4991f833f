"""The dense products at the most rows that their launches take."""
import pytest
import torch

import dense_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,M,N,K", [(torch.bfloat16, 12000000, 1640, 16), (torch.int8, 11625891, 1635, 256)], ids=str)
def test_more_rows_than_small_tiles_take(kind, M, N, K):
    """Results of 38 GB, which more than 2^22 of the tiles that short K is fastest with would make up: first and last rows and columns, and
    rows beside the 32-bit borders of their offsets."""
    from lightop_amd import gemmopt

    print("[case] dense gated", kind, M, N, K, flush=True)
    g = torch.Generator(device="cuda").manual_seed(M)
    _, b, _, sb = ref.operands(kind, 1, 2 * N, K, g)
    if kind == torch.int8:
        a = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device="cuda")
        sa = torch.rand(M, 1, generator=g, device="cuda") * 0.02 + 0.005
        out = gemmopt.gemm_w8a8_act_and_mul(a, b, sa, sb)
    else:
        a, sa = torch.randn(M, K, generator=g, dtype=kind, device="cuda"), None
        out = gemmopt.gemm_act_and_mul(a, b)
    for at in (0, (1 << 31) // N - 50, (1 << 32) // N - 50, M - 100):
        rows = slice(at, at + 100)
        ref.check(out[rows], ref.dense(a[rows], b, None if sa is None else sa[rows], sb, activation="silu", gated=True))
    del a, sa, out
    torch.cuda.empty_cache()
