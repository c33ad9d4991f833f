"""The dense blocks' operators together, as a layer uses them: norms on both sides, router, shared expert, routed experts, a projection."""
import pytest
import torch

import dense_ref as ref
from fp8_ref import ULP32

pytestmark = pytest.mark.gpu


def _layer(M, seed):
    H, I, E = 1024, 512, 8
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")

    def weight(*s):
        return torch.randint(-127, 128, s, generator=g, dtype=torch.int8, device="cuda"), (0.5 + torch.rand(*s[:-1], generator=g, device="cuda")) / (74.0 * s[-1] ** 0.5)

    return dict(x=ref.rows(M, H, g, torch.bfloat16), r=(4 * normal(M, H)).bfloat16(), wo=(normal(H, H) / H ** 0.5).bfloat16(), bo=normal(H).bfloat16(),
                post=(1 + 0.1 * normal(H)).bfloat16(), pre=(1 + 0.1 * normal(H)).bfloat16(), gate=normal(M, 1).bfloat16(),
                router=(normal(E, H) / H ** 0.5).bfloat16(), w13=weight(2 * I, H), w2=weight(H, I), e13=weight(E, 2 * I, H), e2=weight(E, H, I))


def _run(p, cache):
    """Projection with bias -> norms with the residual -> router and shared expert (residual: nothing yet) -> routed experts, the shared expert's output
    added -> norms with the block's gate."""
    from lightop_amd import gemmopt
    from lightop_amd.moe import fused_experts_impl_int8, topk_softmax
    from lightop_amd.norm import rms_norm_block
    from lightop_amd.quant import per_token_quant_int8

    M, k = p["x"].shape[0], 2
    s = {}
    s["attn"] = gemmopt.gemm_bias_act(p["x"], p["wo"], bias=p["bo"])
    s["n"] = rms_norm_block(s["attn"], p["r"], p["pre"], post_weight=p["post"], scale=0.5, quant_dtype=torch.int8, return_normed=True)
    s["logits"] = gemmopt.gemm_bias_act(s["n"].normed, p["router"], out_dtype=torch.float32)
    tw, ids = torch.empty(M, k, device="cuda"), torch.empty(M, k, dtype=torch.int32, device="cuda")
    topk_softmax(tw, ids, None, s["logits"], True)
    s["h"] = gemmopt.gemm_w8a8_act_and_mul(s["n"].q, p["w13"][0], s["n"].scale, p["w13"][1])
    s["q"] = per_token_quant_int8(s["h"])
    s["shared"] = gemmopt.gemm_w8a8_bias_act(s["q"][0], p["w2"][0], s["q"][1], p["w2"][1])
    s["routed"] = fused_experts_impl_int8(s["n"].normed, p["e13"][0], p["e2"][0], tw, ids, cache, use_int8_w8a8=True, per_channel_quant=True,
                                          w1_scale=p["e13"][1].unsqueeze(-1), w2_scale=p["e2"][1].unsqueeze(-1), shared_output=s["shared"])
    s["end"] = rms_norm_block(s["routed"], s["n"].residual, p["pre"], gate=p["gate"], gate_activation="sigmoid")
    # the dense form of the same block: the second product adds the residual itself, in place
    total = s["n"].residual.clone()
    s["dense"] = gemmopt.gemm_w8a8_bias_act(s["q"][0], p["w2"][0], s["q"][1], p["w2"][1], residual=total, out=total)
    s["half"] = gemmopt.gemm_act_and_mul(s["n"].normed, torch.cat([p["wo"], p["wo"].flip(0)]), activation="gelu")
    return s


def _stages(s, p):
    """Each stage against float64 on what the stage before it made."""
    n = s["n"]
    ref.check(s["attn"], ref.dense(p["x"], p["wo"], bias=p["bo"]))
    z = p["r"].double() + 0.5 * _normed(s["attn"].double()) * p["post"].double()
    assert ((n.residual.double() - z).abs() <= 2.0 ** -8 * z.abs() + 64 * ULP32 * (p["r"].double().abs() + z.abs())).all()
    y = _normed(z) * p["pre"].double()
    assert ((n.normed.double() - y).abs() <= 1.01 * 2.0 ** -8 * y.abs() + 1e-5).all()
    assert ((n.q.double() * n.scale.double() - y).abs() <= 0.501 * n.scale.double() + 1e-5).all()
    ref.check(s["logits"], ref.dense(n.normed, p["router"]))
    ref.check(s["h"], ref.dense(n.q, p["w13"][0], n.scale, p["w13"][1], activation="silu", gated=True))
    ref.check(s["shared"], ref.dense(s["q"][0], p["w2"][0], s["q"][1], p["w2"][1]))
    ref.check(s["dense"], ref.dense(s["q"][0], p["w2"][0], s["q"][1], p["w2"][1], residual=n.residual))
    ref.check(s["half"], ref.dense(n.normed, torch.cat([p["wo"], p["wo"].flip(0)]), activation="gelu", gated=True))
    z = n.residual.double() + torch.sigmoid(p["gate"].double()) * s["routed"].double()
    assert ((s["end"].residual.double() - z).abs() <= 1.01 * 2.0 ** -8 * z.abs() + 1e-5).all()


def _normed(v):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6)


@pytest.mark.parametrize("M", [1, 5, 12, 64, 300])
def test_block(M):
    p = _layer(M, M)
    cache = torch.empty(M * 2 * 1024, dtype=torch.bfloat16, device="cuda")
    s = _run(p, cache)
    _stages(s, p)
    same = _run(p, cache)
    assert torch.equal(s["end"].normed, same["end"].normed) and torch.equal(s["dense"], same["dense"])


@pytest.mark.parametrize("M", [1, 64])
def test_captured_block(M):
    """The whole chain in a graph, replayed over other inputs."""
    p = _layer(M, 7)
    cache = torch.empty(M * 2 * 1024, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(p, cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = _run(p, cache)
    for k in range(3):
        other = _layer(M, 8 + k)
        p["x"].copy_(other["x"])
        p["r"].copy_(other["r"])
        graph.replay()
        torch.cuda.synchronize()
        eager = _run(p, torch.empty_like(cache))
        torch.cuda.synchronize()
        for name in ("attn", "logits", "h", "shared", "routed", "dense", "half"):
            assert torch.equal(made[name], eager[name]), name
        assert torch.equal(made["end"].normed, eager["end"].normed) and torch.equal(made["end"].residual, eager["end"].residual)
