"""That the sizes which the GPU tests take for products in parts of K are such.  Host only."""
import pytest

import dense_parts as parts


@pytest.mark.parametrize("size", parts.PARTS, ids=str)
def test_sizes_in_parts(size):
    need = parts.needs(*size)
    kind, M, N, K, gated = size
    tm, tn, n, _ = parts.plan(*size)
    assert need == n * M * ((N + 3) // 4 * 4) * (2 if gated else 1) * 4
    assert parts.plan(*size, workspace=False)[2] == 1


def test_workspaces_of_two_sizes():
    """Among them smaller and larger ones than a stream's workspace begins with (1 MiB)."""
    assert min(parts.needs(*s) for s in parts.PARTS) < 1 << 20 < 2 << 20 < max(parts.needs(*s) for s in parts.PARTS)
