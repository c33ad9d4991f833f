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
