"""e4m3 quantisation of rows, plain and behind a gated activation, against float64."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_sixteen_bit_values_round_right(dtype):
    """Every finite pattern, under maxima of every kind: the codes are the exact quotients', ties to even."""
    from lightop_amd.quant import per_token_group_quant_fp8

    bits = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype).cuda()
    bits = bits[torch.isfinite(bits)]
    g = torch.Generator(device="cuda").manual_seed(1)
    tops = bits[torch.randint(0, bits.numel(), (96,), generator=g, device="cuda")].abs()
    tops = torch.cat([tops, torch.tensor([448, 1, 127, 3.5, 7, 0.875, 255, 257], dtype=dtype, device="cuda")])
    for top in tops:
        v = bits[bits.abs() <= top]
        pad = -v.numel() % 127
        v = torch.cat([v, torch.zeros(pad, dtype=dtype, device="cuda")]).view(-1, 127)
        x = torch.cat([top.expand(v.shape[0], 1), v], dim=1).contiguous()
        q, s = per_token_group_quant_fp8(x, 128, eps=1e-30)
        quotient, scale = ref.groups_fp8(x.double(), 1e-30)
        ok = scale.float() * 448 >= 1e-28  # (a group of nothing but denormal bf16 values)
        assert ((s.double() - scale).abs() <= ref.ULP32 * scale)[ok].all()
        assert torch.equal(q.double()[ok[:, 0]], ref.e4m3(quotient)[ok[:, 0]]), float(top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("M,K", [(1, 128), (1, 7168), (3, 384), (333, 1152), (2000, 2048)])
def test_rows(dtype, M, K):
    from lightop_amd.quant import per_token_group_quant_fp8

    g = torch.Generator(device="cuda").manual_seed(M + K)
    x = ref.rows(M, K, g, "cuda", dtype)
    q, s = per_token_group_quant_fp8(x, 128)
    quotient, scale = ref.groups_fp8(x.double())
    assert ((s.double() - scale).abs() <= ref.ULP32 * scale).all()
    if dtype == torch.float32:  # the quotient is rounded to fp32 first
        assert ref.codes_ok(q, quotient, 2 * ref.ULP32)
    else:
        assert torch.equal(q.double(), ref.e4m3(quotient))


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("M,I", [(1, 128), (5, 768), (333, 1408), (1000, 2048)])
def test_gated(act, dtype, M, I):
    """The activation is a handful of fp32 roundings off (exponential and reciprocal an ulp each, erfc's few): 2^-20 for value and maximum."""
    from lightop_amd.moe import act_and_mul_group_quant_fp8

    g = torch.Generator(device="cuda").manual_seed(M + I)
    x = ref.rows(M, 2 * I, g, "cuda", dtype)
    q, s = act_and_mul_group_quant_fp8(x, act)
    quotient, scale = ref.groups_fp8(ref.act_mul(act, x.double()))
    assert q.shape == (M, I) and ((s.double() - scale).abs() <= 2.0 ** -20 * scale).all()
    assert ref.codes_ok(q, quotient, 2.0 ** -19)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_far_gates(act):
    """Gates down to where the activation ends: relative to the true value, not to the row's largest."""
    from lightop_amd.moe import act_and_mul_group_quant_fp8

    low = -80.0 if act == "silu" else -12.0
    gates = torch.linspace(low, 80, 4096, device="cuda")
    x = torch.zeros(4096, 256, device="cuda")
    x[:, 0] = gates
    x[:, 128] = 1.0
    q, s = act_and_mul_group_quant_fp8(x, act)
    y = ref.act_mul(act, torch.stack([gates.double(), torch.ones_like(gates.double())], -1))[:, 0]
    want = y.abs().clamp(min=1e-10) / 448
    # 0.5 g erfc(-g / sqrt 2): the argument's rounding times its size, 2 (g^2 / 2) 2^-24, on top
    rel = 2.0 ** -20 + (0 if act == "silu" else gates.double().square() * ref.ULP32 * (gates < 0))
    assert ((s[:, 0].double() - want).abs() <= rel * want + 1e-45).all()


def test_zeros_infinities_and_nans():
    from lightop_amd.quant import per_token_group_quant_fp8

    x = torch.ones(5, 256, dtype=torch.bfloat16, device="cuda")
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 3] = float("nan")
    x[3, :128] = -float("inf")
    q, s = per_token_group_quant_fp8(x, 128)
    f = q.float()
    assert (f[0] == 0).all() and torch.equal(s[0], torch.full_like(s[0], 1e-10) / torch.full_like(s[0], 448.0))
    assert s[1, 0].isinf() and f[1, 3].isnan() and (f[1, :3] == 0).all() and (f[1, 128:] == 448).all()
    assert f[2, 3].isnan() and (f[2, :3] == 448).all() and s[2, 0] == 1 / torch.tensor(448.0)
    assert s[3, 0].isinf() and f[3, :128].isnan().all() and (f[3, 128:] == 448).all()


def test_many_rows_strides_and_empties(monkeypatch):
    from lightop_amd import _lib
    from lightop_amd.moe import act_and_mul_group_quant_fp8
    from lightop_amd.quant import per_token_group_quant_fp8

    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1100000, 128, generator=g, device="cuda", dtype=torch.float16)  # more groups than one pass of the largest grid
    q, s = per_token_group_quant_fp8(x, 128)
    for part in (slice(0, 5000), slice(-5000, None)):
        quotient, _ = ref.groups_fp8(x[part].double())
        assert torch.equal(q[part].double(), ref.e4m3(quotient))
    x = torch.randn(6, 2, 512, generator=g, device="cuda")
    want = per_token_group_quant_fp8(x, 128)
    assert want[0].shape == (6, 2, 512) and want[1].shape == (6, 2, 4)
    for y in (x.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([x[:1], x]).view(-1)[1024:].view(6, 2, 512),
              torch.zeros(6 * 1024 + 1, device="cuda")[1:].view(6, 2, 512).copy_(x)):
        got = per_token_group_quant_fp8(y, 128)
        assert torch.equal(got[0].view(torch.int8), want[0].view(torch.int8)) and torch.equal(got[1], want[1])
    gated = act_and_mul_group_quant_fp8(x)
    monkeypatch.setattr(_lib, "_host", _lib._NoHost())
    for a, b in ((per_token_group_quant_fp8(x, 128), want), (act_and_mul_group_quant_fp8(x), gated)):
        assert torch.equal(a[0].view(torch.int8), b[0].view(torch.int8)) and torch.equal(a[1], b[1])
    assert per_token_group_quant_fp8(x[:0], 128)[1].shape == (0, 2, 4)
    assert act_and_mul_group_quant_fp8(x[:0])[0].shape == (0, 2, 256)
    for bad in (lambda: per_token_group_quant_fp8(x.int(), 128), lambda: act_and_mul_group_quant_fp8(x[..., :128]),
                lambda: per_token_group_quant_fp8(x, 128, eps=0.0)):
        with pytest.raises(RuntimeError):
            bad()
