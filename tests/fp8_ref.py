"""The 8-bit operators' definitions in float64, and the bounds that fp32 arithmetic keeps to."""
import torch

G = 128
FP8 = torch.float8_e4m3fn
# Sizes M, N, K of the dense product by the tile they take with a workspace (tokens, columns, whether K is in parts): rows and columns that end
# inside a tile, columns in fours and not, numbers of K blocks that are no multiple of four, more than 64 of them.
TILES = {(64, 32, False): [(17, 21, 384), (100, 700, 1664), (59, 6020, 8320)], (64, 32, True): [(18, 21, 2432), (17, 20, 8320), (130, 300, 7552)],
         (64, 64, False): [(18, 8285, 896), (157, 4356, 8448)], (64, 64, True): [(17, 1461, 6272), (19, 1380, 8320)],
         (128, 128, False): [(197, 8199, 384), (262, 7316, 8576)], (128, 128, True): [(66, 2751, 5760), (67, 2052, 8832)],
         (128, 256, False): [(398, 8273, 384), (409, 8500, 8832)], (128, 256, True): [(18, 5661, 6912), (17, 5780, 8576)],
         (192, 256, False): [(1025, 7291, 384), (1041, 7320, 8576)], (256, 256, False): [(1553, 7255, 384), (1741, 6740, 8448)]}
TILE_SIZES = [(tile, size) for tile in TILES for size in TILES[tile]]
ULP32 = 2.0 ** -24  # one fp32 rounding, relative


def e4m3_step(v):
    """Distance of neighbouring e4m3 values at v (float64)."""
    a = v.abs().clamp(min=2.0 ** -6, max=448.0)
    return (a.view(torch.int64) & 0x7ff0000000000000).view(torch.float64) / 8  # (torch.ldexp goes through an inexact power on the GPU)


def e4m3(v):
    """float64 -> nearest e4m3 value, ties to even, as float64."""
    step = e4m3_step(v)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def groups_fp8(x, eps=1e-10):
    """(quotients 448 v / top, scales) of float64 rows."""
    v = x.unflatten(-1, (-1, G))
    top = v.abs().amax(-1).clamp(min=eps)
    return (448.0 * v / top.unsqueeze(-1)).flatten(-2), top / 448.0


def dequant(q, s):
    return (q.double().unflatten(-1, (-1, G)) * s.double().unsqueeze(-1)).flatten(-2)


def dequant_weight(w, s):
    rows = s.double().repeat_interleave(G, dim=-2).narrow(-2, 0, w.shape[-2])
    return dequant(w, rows)


def act_mul(name, h):
    g, u = h.chunk(2, dim=-1)
    a = g * torch.sigmoid(g) if name == "silu" else 0.5 * g * torch.erfc(g * -(0.5 ** 0.5))
    return a * u


def codes_ok(q, quotient, rel):
    """Codes are the nearest to quotients that are off by `rel` at most (saturating at 448)."""
    off = (q.double() - quotient).abs()
    return bool((off <= 0.5 * e4m3_step(quotient) + rel * quotient.abs() + 1e-12).all())


def half_step(dtype, v):
    """Half a step of the output type at v, and of its smallest number."""
    f = torch.finfo(dtype)
    return v.abs() * (f.eps / 2) + f.tiny * f.eps


def weights(shape, g, dev, scale=2e-4):
    w = (torch.randn(shape, generator=g, device=dev) * 100).clamp(-448, 448).to(FP8)
    s = torch.exp(0.3 * torch.randn(shape[:-2] + (-(-shape[-2] // G), shape[-1] // G), generator=g, device=dev)) * scale
    return w, s


def rows(M, K, g, dev, dtype=torch.float32):
    x = torch.randn(M, K, generator=g, device=dev)
    x[:, ::64] *= 8
    return x.to(dtype)
