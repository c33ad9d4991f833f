"""The dense blocks' operators in float64, and the bounds that fp32 arithmetic keeps to."""
import torch

from fp8_ref import ULP32, half_step

SILU_SLOPE, GELU_SLOPE = 1.1, 1.13  # largest derivatives: 1.0998 and 1.1290


def rows(M, K, g, dtype):
    """Activations: unit normal, one channel in 64 eight times as wide."""
    x = torch.randn(M, K, generator=g, dtype=torch.float32, device="cuda")
    x[:, ::64] *= 8.0
    return x.to(dtype)


def operands(kind, M, N, K, g):
    """a, b, a_scale, b_scale (None with 16 bits); ``kind``: torch.bfloat16, torch.float16 or torch.int8."""
    if kind != torch.int8:
        return rows(M, K, g, kind), (torch.randn(N, K, generator=g, dtype=torch.float32, device="cuda") / K ** 0.5).to(kind), None, None
    a = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device="cuda")
    b = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8, device="cuda")
    sa = torch.rand(M, 1, generator=g, device="cuda") * 0.02 + 0.005
    sb = (torch.rand(N, generator=g, device="cuda") + 0.2) / (74.0 * K ** 0.5)
    return a, b, sa, sb


def act(name, v):
    if name is None:
        return v
    return v * torch.sigmoid(v) if name == "silu" else 0.5 * v * torch.erfc(v * -(0.5 ** 0.5))


def dense(a, b, sa=None, sb=None, bias=None, activation=None, gated=False, residual=None, scale=1.0):
    """(exact result, bound of an fp32 evaluation before the result's rounding).

    A matrix instruction adds 32 products of 16-bit values (exact in fp32) to the sum, in steps of which each may cut off an fp32 ulp
    (2 ** -23): K / 32 instructions and 32 products deep, and 8 parts of K at the most.  An int8 sum is exact."""
    ad, bd = a.double(), b.double()
    v = ad @ bd.T
    if sa is not None:
        both = sa.double().reshape(-1, 1) * sb.double().reshape(1, -1)
        v = v * both
        off = 3 * ULP32 * v.abs()
    else:
        off = (a.shape[1] // 32 + 1 + 32 + 8) * 2 * ULP32 * (ad.abs() @ bd.abs().T)
    if bias is not None:
        v = v + bias.double()
    off = off + 2 * ULP32 * v.abs()
    slope, tail = {None: (1.0, 0.0), "silu": (SILU_SLOPE, 8 * ULP32), "gelu": (GELU_SLOPE, 16 * ULP32)}[activation]
    if gated:
        g, u = v.chunk(2, dim=-1)
        og, ou = off.chunk(2, dim=-1)
        y = act(activation, g) * u
        off = (act(activation, g).abs() + slope * og) * ou + u.abs() * (slope * og + tail * g.abs()) + ULP32 * y.abs()
    else:
        y = act(activation, v)
        off = slope * off + tail * v.abs()
    y, off = y * scale, off * abs(scale) + 2 * ULP32 * (y * scale).abs()
    if residual is not None:
        y = y + residual.double()
        off = off + ULP32 * y.abs()
    return y, off


def check(out, want):
    exact, off = want
    assert out.shape == exact.shape
    bad = ~((out.double() - exact).abs() <= off * 1.01 + 1.01 * half_step(out.dtype, exact) + 1e-30)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


# Sizes M, N, K (16-bit operands; int8 ones of twice the K take the same) by the tile they take with a workspace: (tokens, weight rows, whether K is in parts, gated).
# Rows and columns end inside a tile, K inside a K block; the first N is a multiple of eight, the second odd.
TILES = {
    (32, 32, False, False): [(12, 16, 208), (9, 21, 224)],
    (32, 32, False, True): [(9, 24, 232), (11, 17, 224)],
    (32, 32, True, False): [(9, 16, 2216), (9, 17, 2256)],
    (32, 32, True, True): [(9, 24, 2456), (9, 17, 2336)],
    (64, 32, False, False): [(1652, 136, 232), (34, 4497, 264)],
    (64, 32, False, True): [(45, 2248, 208), (33, 2147, 224)],
    (64, 32, True, False): [(2084, 16, 5216), (1083, 33, 4912)],
    (64, 32, True, True): [(1046, 40, 4568), (1059, 17, 5200)],
    (64, 64, False, False): [(69, 5704, 200), (35, 8633, 264)],
    (64, 64, False, True): [(18, 8584, 248), (19, 8377, 224)],
    (64, 64, True, False): [(34, 1512, 3984), (1361, 33, 3680)],
    (64, 64, True, True): [(35, 696, 4208), (34, 677, 3472)],
    (64, 128, False, False): [(268, 3760, 264), (77, 8677, 280)],
    (64, 128, False, True): [(21, 8560, 432), (19, 8193, 296)],
    (64, 128, True, False): [(17, 8248, 2480), (17, 8363, 2664)],
    (64, 128, True, True): [(17, 4184, 2824), (18, 4383, 2600)],
    (96, 96, False, False): [(1491, 1456, 200), (399, 5099, 200)],
    (96, 96, False, True): [(68, 8336, 208), (93, 8371, 216)],
    (96, 96, True, False): [(68, 3216, 4216), (68, 2769, 3344)],
    (96, 96, True, True): [(71, 1520, 3624), (65, 1401, 3352)],
    (128, 128, False, False): [(473, 5080, 336), (208, 8581, 368)],
    (128, 128, False, True): [(130, 7608, 360), (102, 8621, 368)],
    (128, 128, True, False): [(65, 8392, 3336), (69, 8297, 2872)],
    (128, 128, True, True): [(67, 4272, 3480), (66, 4329, 3112)],
    (128, 192, False, False): [(542, 8376, 208), (1155, 3917, 200)],
    (128, 192, False, True): [(220, 8936, 200), (484, 4247, 216)],
    (128, 192, True, False): [(397, 2768, 4656), (291, 3591, 4040)],
    (128, 192, True, True): [(98, 5624, 4072), (100, 5555, 4024)],
    (128, 256, False, False): [(819, 7056, 208), (702, 8209, 208)],
    (128, 256, False, True): [(676, 4184, 208), (521, 4919, 200)],
    (192, 256, False, False): [(1029, 8984, 280), (1088, 8509, 200)],
    (192, 256, False, True): [(1184, 3984, 200), (1860, 2489, 200)],
    (256, 256, False, False): [(2325, 5104, 216), (1617, 7551, 200)],
    (256, 256, False, True): [(1439, 4464, 208), (2309, 2603, 200)],
}
TILE_SIZES = [(tile, size) for tile in TILES for size in TILES[tile]]
