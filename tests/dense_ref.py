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
    (32, 32, False, False): [(11, 16, 408), (10, 17, 360)],
    (32, 32, False, True): [(10, 24, 328), (10, 19, 352)],
    (32, 32, True, False): [(9, 16, 2488), (9, 17, 2504)],
    (32, 32, True, True): [(9, 24, 2456), (9, 17, 2416)],
    (64, 32, False, False): [(12, 16, 208), (9, 21, 224)],
    (64, 32, False, True): [(9, 24, 232), (11, 17, 224)],
    (64, 32, True, False): [(1356, 40, 3040), (1381, 33, 3104)],
    (64, 32, True, True): [(35, 696, 3064), (1370, 17, 3040)],
    (64, 64, False, False): [(47, 8520, 328), (33, 8695, 328)],
    (64, 64, False, True): [(67, 3280, 360), (39, 4285, 376)],
    (64, 64, True, False): [(33, 4256, 2776), (33, 4207, 2784)],
    (64, 64, True, True): [(34, 2120, 2832), (35, 2119, 2776)],
    (64, 128, False, False): [(153, 6328, 216), (149, 6139, 200)],
    (64, 128, False, True): [(12, 8568, 288), (9, 8545, 224)],
    (64, 128, True, False): [(9, 8416, 2792), (9, 8307, 2376)],
    (64, 128, True, True): [(9, 2088, 5280), (9, 4243, 2336)],
    (96, 96, False, False): [(1491, 1456, 200), (602, 3363, 208)],
    (96, 96, False, True): [(68, 8336, 208), (93, 8371, 216)],
    (96, 96, True, False): [(68, 3216, 4216), (65, 2757, 4704)],
    (96, 96, True, True): [(77, 1376, 4408), (65, 1491, 4184)],
    (128, 128, False, False): [(223, 8256, 248), (399, 5099, 200)],
    (128, 128, False, True): [(203, 4144, 232), (199, 4685, 208)],
    (128, 128, True, False): [(67, 4424, 4920), (66, 8217, 2408)],
    (128, 128, True, True): [(65, 3168, 4336), (65, 4327, 2096)],
    (128, 192, False, False): [(542, 8376, 208), (1155, 3917, 200)],
    (128, 192, False, True): [(220, 8936, 200), (484, 4247, 216)],
    (128, 192, True, False): [(141, 5992, 5512), (133, 5549, 4856)],
    (128, 192, True, True): [(10, 5488, 4144), (9, 5917, 3728)],
    (128, 256, False, False): [(819, 7056, 208), (702, 8209, 208)],
    (128, 256, False, True): [(676, 4184, 208), (521, 4919, 200)],
    (128, 256, True, True): [(9, 8200, 4176), (10, 8275, 4056)],
    (192, 256, False, False): [(1045, 7456, 208), (946, 8195, 200)],
    (192, 256, False, True): [(1184, 3984, 200), (391, 8271, 208)],
    (256, 256, False, False): [(2325, 5104, 216), (1617, 7551, 200)],
    (256, 256, False, True): [(1009, 5552, 208), (2309, 2603, 200)],
}
TILE_SIZES = [(tile, size) for tile in TILES for size in TILES[tile]]
