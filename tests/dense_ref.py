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
    (32, 32, False, False): [(18, 16, 336), (20, 19, 352)],
    (32, 32, False, True): [(17, 24, 360), (17, 17, 376)],
    (32, 32, True, False): [(7, 16, 5448), (7, 17, 5480)],
    (32, 32, True, True): [(11, 24, 3464), (7, 17, 5448)],
    (64, 32, False, False): [(28, 16, 224), (17, 23, 200)],
    (64, 32, False, True): [(20, 24, 200), (18, 19, 216)],
    (64, 32, True, False): [(1356, 40, 3040), (1381, 33, 3104)],
    (64, 32, True, True): [(35, 696, 3064), (1370, 17, 3040)],
    (64, 64, False, False): [(47, 8520, 328), (33, 8695, 328)],
    (64, 64, False, True): [(67, 3280, 360), (39, 4285, 376)],
    (64, 64, True, False): [(33, 4256, 2776), (33, 4207, 2784)],
    (64, 64, True, True): [(34, 2120, 2832), (35, 2119, 2776)],
    (64, 128, False, False): [(153, 6328, 216), (149, 6139, 200)],
    (64, 128, False, True): [(18, 8664, 496), (18, 8529, 200)],
    (64, 128, True, False): [(17, 8568, 2928), (17, 8549, 2376)],
    (64, 128, True, True): [(18, 4528, 2488), (19, 4103, 2464)],
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
    (128, 192, True, True): [(17, 5536, 4072), (18, 5473, 4440)],
    (128, 256, False, False): [(819, 7056, 208), (702, 8209, 208)],
    (128, 256, False, True): [(676, 4184, 208), (521, 4919, 200)],
    (128, 256, True, True): [(18, 8416, 4432), (17, 8737, 4048)],
    (192, 256, False, False): [(1045, 7456, 208), (946, 8195, 200)],
    (192, 256, False, True): [(1184, 3984, 200), (391, 8271, 208)],
    (256, 256, False, False): [(2325, 5104, 216), (1617, 7551, 200)],
    (256, 256, False, True): [(1009, 5552, 208), (2309, 2603, 200)],
}
TILE_SIZES = [(tile, size) for tile in TILES for size in TILES[tile]]

# Sizes M, N, K, gated of up to 16 tokens, one for every C, number of waves and U of their kernel; columns and K end inside a workgroup's part and a K block.
FEW = [
    (16, 5, 24, False), (16, 8184, 72, False), (16, 8515, 136, False), (16, 4108, 200, True), (16, 8184, 272, False), (16, 8238, 328, False), (8, 5, 392, True), (16, 8598, 472, False),
    (16, 5, 72, False), (16, 5, 136, False), (16, 5, 264, True), (16, 5, 392, True), (16, 5, 520, True), (16, 5, 656, True), (16, 5, 776, True), (16, 5, 904, True),
    (16, 5, 200, False), (16, 5, 264, False), (16, 5, 520, False), (16, 5, 784, False), (16, 5, 1032, False), (16, 5, 1312, False), (16, 5, 1552, False), (16, 5, 1824, False),
    (16, 5, 2256, False), (8, 17355, 456, False), (8, 6219, 464, True), (8, 9, 456, False), (8, 9, 520, False), (8, 9, 648, False), (8, 9, 784, False), (8, 4125, 904, False),
    (8, 8209, 464, False), (5, 4106, 1184, False), (8, 9, 920, False), (8, 9, 1040, False), (8, 9, 1312, False), (8, 9, 1552, False), (8, 9, 1816, False), (8, 9, 2456, False),
    (8, 9, 2592, False), (8, 9, 3120, False), (8, 9, 3624, False), (8, 9, 4512, False), (4, 8210, 1000, False), (4, 3075, 992, True), (4, 5, 984, False), (4, 5, 1032, False),
    (4, 5, 1304, False), (4, 5, 1568, False), (4, 1053, 1848, True), (4, 4119, 1008, False), (4, 1047, 2352, True), (4, 5, 1800, False), (4, 5, 2056, False), (4, 5, 2568, False),
    (4, 5, 3144, False), (4, 5, 3600, False), (4, 5, 4896, False), (4, 5, 5304, False), (4, 5, 6152, False), (4, 5, 7216, False), (4, 5, 8968, False), (2, 2132, 2032, True),
    (2, 1540, 2032, True), (2, 5, 2000, False), (2, 5, 2056, False), (2, 5, 2568, False), (2, 5, 3080, False), (2, 521, 3696, True), (2, 1036, 1992, True), (2, 1033, 4616, False),
    (2, 5, 3688, False), (2, 5, 4128, False), (2, 5, 5160, False), (2, 5, 6216, False), (2, 5, 7280, False), (2, 5, 10024, False), (2, 5, 10248, False), (2, 5, 12328, False),
    (2, 5, 14344, False), (1, 2097, 4088, False), (1, 1538, 4072, False), (1, 5, 4080, False), (1, 5, 4104, False), (1, 5, 5128, False), (1, 5, 6280, False), (1, 515, 7176, False),
    (1, 1062, 4080, False), (1, 527, 9296, False), (1, 5, 7368, False), (1, 5, 8216, False), (1, 5, 10296, False), (1, 5, 12576, False), (1, 5, 14360, False),
]
