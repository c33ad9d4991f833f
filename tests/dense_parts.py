"""Sizes of the dense products whose K is taken in parts, which go through a workspace and a joining launch."""
import ctypes

import torch

CODES = {torch.bfloat16: 0, torch.float16: 1, torch.int8: 3}

# operands' type, tokens, columns of the result, K, gated
PARTS = [(torch.bfloat16, 20, 576, 7168, False), (torch.float16, 333, 577, 7168, False), (torch.int8, 20, 288, 7168, True), (torch.int8, 130, 300, 16384, False),
         (torch.bfloat16, 333, 289, 7168, True), (torch.float16, 70, 250, 7160, False), (torch.int8, 33, 131, 14320, False), (torch.bfloat16, 17, 131, 7160, True)]


def plan(kind, M, N, K, gated, workspace=True):
    """(tile's tokens, tile's weight rows, parts of K, bytes of workspace) of a call."""
    from lightop_amd import _lib

    lib, at = _lib.lib(), [ctypes.c_int32() for _ in range(3)]
    assert lib.lo_gemm_bias_act_tile_query(CODES[kind], int(gated), M, N, K, int(workspace), *(ctypes.byref(v) for v in at)) == 0
    return tuple(v.value for v in at) + (lib.lo_gemm_bias_act_workspace_bytes(CODES[kind], int(gated), M, N, K),)


def needs(kind, M, N, K, gated):
    """Bytes of the workspace of a size that has to be split."""
    _, _, parts, need = plan(kind, M, N, K, gated)
    assert parts > 1 and need > 0, (kind, M, N, K, gated)
    return need

# Sizes M, N, K (16-bit operands; int8 ones of twice the K take the same) of plain products on tiles of 128 x 256 in parts; columns and K end inside a tile and a K block.
WIDE = [(18, 18024, 4392), (17, 16969, 5360), (175, 9125, 10984)]
