"""The 8-bit operators' definitions in float64, and the bounds that fp32 arithmetic keeps to."""
import torch

G = 128
FP8 = torch.float8_e4m3fn
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
