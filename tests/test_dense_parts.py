"""That the sizes which the GPU tests take for products in parts of K are such.  Host only."""
import random

import pytest
import torch

import dense_parts as parts
import dense_ref as ref


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


@pytest.mark.parametrize("M,N,K", parts.WIDE)
def test_sizes_of_wide_tiles_in_parts(M, N, K):
    for kind, k in ((torch.bfloat16, K), (torch.float16, K), (torch.int8, 2 * K)):
        tm, tn, n, need = parts.plan(kind, M, N, k, False)
        assert (tm, tn) == (128, 256) and n > 1 and need > 0


def test_no_form_is_without_sizes():
    """Whatever a call takes, whole or in parts, plain or gated, is among the sizes that the GPU tests run: over a grid and over random sizes."""
    covered = set(ref.TILES) | {(128, 256, True, False), (16, 16, False, False), (16, 16, False, True)}
    rng, seen = random.Random(5), set()
    sizes = [(M, N, K) for M in (1, 9, 17, 33, 65, 200, 800, 3200, 8000) for N in (16, 130, 577, 2000, 8000, 18000) for K in (16, 208, 1008, 4000, 8000, 15008)]
    sizes += [(int(2 ** rng.uniform(0, 14)), int(2 ** rng.uniform(0, 17)), 16 * int(2 ** rng.uniform(0, 10))) for _ in range(20000)]
    for M, N, K in sizes:
        kind, gated = rng.choice((torch.bfloat16, torch.float16, torch.int8)), rng.random() < 0.4
        tm, tn, n, _ = parts.plan(kind, M, N, K, gated)
        seen.add((tm, tn, n > 1, gated))
    assert seen <= covered and (128, 256, True, False) in seen
