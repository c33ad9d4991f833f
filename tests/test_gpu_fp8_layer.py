"""The 8-bit operators together, as a layer uses them: norm, shared expert in e4m3, routed experts of either type."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 7, 64])
def test_fp8_layer(M):
    """norm -> codes -> shared expert -> its output into the routed experts; against the same chain in float64 on the codes that each stage
    made (a stage is held to its own bounds elsewhere)."""
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block
    from lightop_amd.moe import act_and_mul_group_quant_fp8, fused_experts_decode_fp8, topk_softmax
    from lightop_amd.norm import rms_norm_quant
    from lightop_amd.quant import per_token_group_quant_fp8

    H, I, E, k = 1024, 512, 8, 2
    g = torch.Generator(device="cuda").manual_seed(M)
    x, res = ref.rows(M, H, g, "cuda", torch.bfloat16), ref.rows(M, H, g, "cuda", torch.bfloat16)
    w = torch.ones(H, device="cuda")
    gate = torch.randn(H, E, generator=g, device="cuda").to(torch.bfloat16)
    sw1, ss1 = ref.weights((2 * I, H), g, "cuda")
    sw2, ss2 = ref.weights((H, I), g, "cuda")
    w1, s1 = ref.weights((E, 2 * I, H), g, "cuda")
    w2, s2 = ref.weights((E, H, I), g, "cuda")

    n = rms_norm_quant(x, w, residual=res, quant_dtype=ref.FP8, group_size=128, return_normed=True)
    h = gemm_w8a8_fp8_block(n.q, sw1, n.scale, ss1)
    aq, a_s = act_and_mul_group_quant_fp8(h)
    shared = gemm_w8a8_fp8_block(aq, sw2, a_s, ss2)
    tw, ids = torch.empty(M, k, device="cuda"), torch.empty(M, k, dtype=torch.int32, device="cuda")
    topk_softmax(tw, ids, None, n.normed @ gate, True)
    out = fused_experts_decode_fp8(n.normed, w1, w2, tw, ids, s1, s2, routed_scaling_factor=2.5, shared_output=shared)

    hd = ref.dequant(n.q, n.scale) @ ref.dequant_weight(sw1, ss1).T
    assert ((h.double() - hd).norm() <= 2.0 ** -8 * hd.norm())
    sd = ref.dequant(aq, a_s) @ ref.dequant_weight(sw2, ss2).T
    assert ((shared.double() - sd).norm() <= 2.0 ** -8 * sd.norm())
    want = shared.double()
    nq, ns = per_token_group_quant_fp8(n.normed, 128)
    rows = ref.dequant(nq, ns)
    for t in range(M):
        for j in range(k):
            e = int(ids[t, j])
            v = ref.act_mul("silu", rows[t] @ ref.dequant_weight(w1[e], s1[e]).T)
            q, s = ref.groups_fp8(v)
            want[t] += 2.5 * float(tw[t, j]) * (ref.dequant(ref.e4m3(q), s) @ ref.dequant_weight(w2[e], s2[e]).T)
    # half a bf16 step, and a code in a thousand a step off
    assert ((out.double() - want).norm() <= (2.0 ** -8 + 2.0 ** -8) * want.norm())


def test_norm_in_front_of_the_int8_experts(monkeypatch):
    """int8 rows of the norm as the per-channel experts' i_q / i_s: what the layer makes of the same codes through its stages."""
    from lightop_amd import workloads as wl
    from lightop_amd.moe import fused_experts_impl_int8
    from lightop_amd.norm import rms_norm_quant
    from lightop_amd.quant import per_token_quant_int8

    monkeypatch.setenv("LMSLIM_USE_FUSED_RMS_QUANT", "1")
    layer = wl.TINY_PC
    w1, w2, s1, s2 = wl.make_weights(layer, seed=0, device="cuda")
    x, tw, ids = (t.cuda() for t in wl.make_inputs(layer, 33, seed=1))
    n = rms_norm_quant(x, torch.ones(layer.H, device="cuda"), residual=x, return_normed=True)
    cache = torch.empty(33 * layer.top_k * max(2 * layer.I, layer.H), dtype=x.dtype, device="cuda")
    call = lambda rows, q, s: fused_experts_impl_int8(rows, w1, w2, tw, ids, cache, use_int8_w8a8=True, per_channel_quant=True, w1_scale=s1,
                                                      w2_scale=s2, i_q=q, i_s=s)
    out = call(n.normed, n.q, n.scale)
    # codes of the rounded rows in their place: a code of the fp32 row is another one where the rounding crosses a border
    q, s = per_token_quant_int8(n.normed)
    near = call(n.normed, q, s)
    assert (n.q != q).float().mean() < 0.2 and (n.q.int() - q.int()).abs().max() <= 1
    assert (out.double() - near.double()).norm() <= 0.02 * near.double().norm()
    assert torch.equal(out, call(torch.zeros_like(x), n.q, n.scale))  # the rows themselves are not read
