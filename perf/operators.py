"""The 8-bit operators around the routed experts, as cases to measure.

Four operators: the RMS norm in front of a layer with its 8-bit output (``rms_norm_quant``), the e4m3
quantisation of rows, plain or behind a gated activation (``per_token_group_quant_fp8``,
``act_and_mul_group_quant_fp8``), the dense product of e4m3 operands with a scale for each block of 128
(``gemm_w8a8_fp8_block``) and the experts of a few tokens with such weights (``fused_experts_decode_fp8``).
Hidden and intermediate sizes are those of ``lightop_amd.workloads``; token counts run from one (a
sequence decoding) to a prefill batch of 8192.

int8 codes come back as bfloat16, which holds them exactly, next to their scales; e4m3 codes as the
floating values they are.
"""
from __future__ import annotations

import math

import torch

#: True: ``run`` makes the calls of the package; False: the plain form in elementary torch operations.
own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
FP8 = torch.float8_e4m3fn
G = 128

# name -> experts on this GPU, experts routed over, top_k, H, I
LAYERS = {"tiny-e8": (8, 8, 2, 1024, 512), "qwen3-30b-a3b": (128, 128, 8, 2048, 768),
          "deepseek-v3-ep8-share": (32, 256, 8, 7168, 2048)}

MAX_TOKENS = 8192
MAX_PRODUCT = 8192 * 4096 * 7168


def _norm(tokens, hidden, form, dtype, residual, normed):
    return {"op": "norm", "tokens": tokens, "hidden": hidden, "form": form, "dtype": dtype, "residual": residual, "normed": normed}


def _quant(tokens, cols, activation, dtype):
    return {"op": "quant", "tokens": tokens, "cols": cols, "activation": activation, "dtype": dtype}


def _gemm(tokens, n, k, dtype):
    return {"op": "gemm", "tokens": tokens, "n": n, "k": k, "dtype": dtype}


def _experts(tokens, layer, activation, dtype, shared):
    return {"op": "experts", "tokens": tokens, "layer": layer, "activation": activation, "dtype": dtype, "shared": shared}


def listed():
    return [
        # one sequence decoding: the rows that the per-channel experts take as i_q, i_s
        dict(_norm(1, 2048, "int8 rows", "bf16", True, False), name="norm, int8 rows, 1"),
        # a chunk of prefill in half precision; the router reads the normed rows too
        dict(_norm(700, 4096, "int8 groups", "fp16", True, True), name="norm, int8 groups, 700"),
        # the largest prefill batch in front of an fp8 layer
        dict(_norm(8192, 7168, "fp8 groups", "bf16", True, False), name="norm, fp8 groups, 8192"),
        # rows of a projection's input
        dict(_quant(333, 7168, "none", "bf16"), name="quant, rows 333"),
        # between the two products of a shared expert
        dict(_quant(4096, 2048, "silu", "bf16"), name="quant, silu 4096"),
        # shared expert of one sequence decoding: gate and up
        dict(_gemm(1, 4096, 7168, "bf16"), name="gemm, decode 1"),
        # the down product of a decode batch
        dict(_gemm(48, 7168, 2048, "bf16"), name="gemm, decode 48"),
        # a narrow projection (neither side a multiple of a tile) of a short chunk
        dict(_gemm(333, 576, 7168, "fp16"), name="gemm, narrow 333"),
        # a chunk of prefill with decode tokens riding along
        dict(_gemm(1531, 7168, 2048, "bf16"), name="gemm, chunk 1531"),
        # the largest prefill batch
        dict(_gemm(8192, 4096, 7168, "bf16"), name="gemm, prefill 8192"),
        # the routed experts of one sequence decoding
        dict(_experts(1, "qwen3-30b-a3b", "silu", "bf16", False), name="experts, decode 1"),
        # a decode batch on an expert-parallel rank, the shared expert's output added
        dict(_experts(24, "deepseek-v3-ep8-share", "silu", "bf16", True), name="experts, rank of 8, 24"),
    ]


def draw(rng):
    def tokens(most):
        return min(most, max(1, round(math.exp(rng.uniform(0.0, math.log(most + 1))))))

    op = rng.choice(("norm", "quant", "gemm", "experts"))
    if op == "norm":
        hidden = rng.choice((1024, 2048, 4096, 7168, G * rng.randint(1, 56)))
        return _norm(tokens(MAX_TOKENS), hidden, rng.choice(("int8 rows", "int8 groups", "fp8 groups")),
                     rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.random() < 0.75, rng.random() < 0.4)
    if op == "quant":
        cols = rng.choice((768, 2048, 4096, 7168, G * rng.randint(1, 56)))
        act = rng.choice(("none", "silu", "gelu"))
        return _quant(tokens(MAX_TOKENS), min(cols, 4096) if act != "none" else cols, act, rng.choice(("bf16", "bf16", "fp16", "fp32")))
    if op == "gemm":
        n, k = rng.choice(((4096, 7168), (7168, 2048), (1536, 2048), (2048, 768), (576, 7168),
                           (rng.randint(1, 7168), G * rng.randint(1, 56))))
        most = max(1, min(MAX_TOKENS, MAX_PRODUCT // (n * k)))
        return _gemm(tokens(most), n, k, rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32")))
    return _experts(tokens(64), rng.choice(tuple(LAYERS)), rng.choice(("silu", "silu", "silu", "gelu")),
                    rng.choice(("bf16", "bf16", "fp16")), rng.random() < 0.5)


def _rows(g, rows, cols, dtype):
    """Activations: unit normal, one channel in 64 eight times as wide, as hidden states have them."""
    x = torch.randn(rows, cols, generator=g, dtype=torch.float32, device=g.device)
    x[:, ::64] *= 8.0
    return x.to(dtype)


def _weights(g, *shape):
    """e4m3 codes of weights whose block maxima are near the type's, and their blocks' scales."""
    w = torch.randn(*shape, generator=g, dtype=torch.bfloat16, device=g.device).mul_(100.0).clamp_(-448.0, 448.0).to(FP8)
    s = torch.randn(*shape[:-2], -(-shape[-2] // G), shape[-1] // G, generator=g, dtype=torch.float32, device=g.device)
    return w, torch.exp(0.3 * s + math.log(2e-4))


def prepare(case, seed):
    dev, M = torch.device("cuda:0"), int(case["tokens"])
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + M)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "norm":
        H = case["hidden"]
        s["x"] = _rows(g, M, H, dtype)
        s["residual"] = (4.0 * _rows(g, M, H, torch.float32)).to(dtype) if case["residual"] else None
        s["weight"] = (1.0 + 0.2 * torch.randn(H, generator=g, dtype=torch.float32, device=dev)).to(dtype)
    elif case["op"] == "quant":
        s["x"] = _rows(g, M, case["cols"] * (1 if case["activation"] == "none" else 2), dtype)
    elif case["op"] == "gemm":
        rows = _rows(g, M, case["k"], torch.float32).view(M, -1, G)
        s["a_scale"] = rows.abs().amax(-1).clamp(min=1e-10) / 448.0
        s["a"] = (rows / s["a_scale"].unsqueeze(-1)).view(M, -1).to(FP8)
        s["b"], s["b_scale"] = _weights(g, case["n"], case["k"])
    else:
        E, Eg, k, H, I = LAYERS[case["layer"]]
        s["x"] = _rows(g, M, H, dtype)
        s["w1"], s["w1_scale"] = _weights(g, E, 2 * I, H)
        s["w2"], s["w2_scale"] = _weights(g, E, H, I)
        p = torch.softmax(torch.randn(M, Eg, generator=g, dtype=torch.float32, device=dev), dim=-1)
        weights, ids = torch.topk(p, k, dim=-1)
        s["weights"], s["ids"] = weights / weights.sum(-1, keepdim=True), ids.to(torch.int32)
        s["map"] = None
        if E < Eg:
            s["map"] = torch.full((Eg,), -1, dtype=torch.int32, device=dev)
            s["map"][:E] = torch.arange(E, dtype=torch.int32, device=dev)
        s["shared"] = _rows(g, M, H, dtype) if case["shared"] else None
        s["factor"] = 2.5 if case["layer"].startswith("deepseek") else 1.0
    return s


# ---- the plain forms: torch.float32 between the inputs and one rounding of each output ----------------------------

def _activate(name, h):
    g, u = h.chunk(2, dim=-1)
    if name == "silu":
        return g / (1.0 + torch.exp(-g)) * u
    return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5))) * u


def _groups(y):
    """Scales and quotients of the e4m3 rule, one scale for 128 values: amax / 448 and 448 y / amax.  The quotients of
    16-bit values are often halfway between two codes; 7/8 y is exact for them, so the division rounds once."""
    v = y.unflatten(-1, (-1, G))
    amax = v.abs().amax(-1).clamp(min=1e-10)
    return (v * 0.875 / (amax / 512.0).unsqueeze(-1)).flatten(-2), amax / 448.0


def _unpack(q, s):
    """The values that e4m3 codes and their groups' scales stand for."""
    return (q.float().unflatten(-1, (-1, G)) * s.unsqueeze(-1)).flatten(-2)


def _unpack_weights(w, s):
    rows = s.repeat_interleave(G, dim=-2).narrow(-2, 0, w.shape[-2])
    return (w.float().unflatten(-1, (-1, G)) * rows.unsqueeze(-1)).flatten(-2)


def _plain_norm(s):
    c = s["case"]
    z = s["x"].float()
    out = {}
    if s["residual"] is not None:
        z = z + s["residual"].float()
        out["residual"] = z.to(s["x"].dtype)
    y = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    if c["normed"]:
        out["normed"] = y.to(s["x"].dtype)
    if c["form"] == "int8 rows":
        amax = y.abs().amax(-1, keepdim=True).clamp(min=1e-10)
        out["scale"] = amax / 127.0
        out["q"] = torch.round(y * (127.0 / amax)).clamp(-128, 127).to(torch.bfloat16)
    elif c["form"] == "int8 groups":
        v = y.unflatten(-1, (-1, G))
        out["scale"] = v.abs().amax(-1).clamp(min=1e-10) / 127.0
        out["q"] = torch.trunc((v / out["scale"].unsqueeze(-1)).clamp(-128, 127)).flatten(-2).to(torch.bfloat16)
    else:
        q, out["scale"] = _groups(y)
        out["q"] = q.to(FP8)
    return out


def _plain_quant(s):
    x = s["x"].float()
    q, scale = _groups(x if s["case"]["activation"] == "none" else _activate(s["case"]["activation"], x))
    return {"q": q.to(FP8), "scale": scale}


def _plain_gemm(s):
    a, b = _unpack(s["a"], s["a_scale"]), _unpack_weights(s["b"], s["b_scale"])
    return {"out": torch.matmul(a, b.t()).to(DTYPES[s["case"]["dtype"]])}


def _plain_experts(s):
    x, (E, M) = s["x"], (s["w1"].shape[0], s["x"].shape[0])
    q, scale = _groups(x.float())
    rows = _unpack(q.to(FP8), scale)
    w1, w2 = _unpack_weights(s["w1"], s["w1_scale"]), _unpack_weights(s["w2"], s["w2_scale"])
    h = torch.matmul(w1.flatten(0, 1), rows.t().contiguous()).view(E, -1, M).transpose(1, 2)
    q, scale = _groups(_activate(s["case"]["activation"], h))
    y = torch.bmm(w2, _unpack(q.to(FP8), scale).transpose(1, 2).contiguous())  # [E, H, M]
    ids = s["ids"].long() if s["map"] is None else s["map"].long()[s["ids"].long()]
    share = torch.zeros(M, E + 1, dtype=torch.float32, device=x.device)  # the last column: experts of other ranks
    share.scatter_add_(1, torch.where(ids < 0, E, ids), s["weights"])
    out = s["factor"] * (y * share[:, :E].t().unsqueeze(1)).sum(0).t()
    if s["shared"] is not None:
        out = out + s["shared"].float()
    return {"out": out.to(x.dtype)}


# ---- the package's calls --------------------------------------------------------------------------------------------

def _own_norm(s):
    from lightop_amd.norm import rms_norm_quant

    c = s["case"]
    r = rms_norm_quant(s["x"], s["weight"], 1e-6, residual=s["residual"], quant_dtype=FP8 if c["form"] == "fp8 groups" else torch.int8,
                       group_size=None if c["form"] == "int8 rows" else G, return_normed=c["normed"])
    out = {"q": r.q if c["form"] == "fp8 groups" else r.q.to(torch.bfloat16), "scale": r.scale}
    if r.residual is not None:
        out["residual"] = r.residual
    if c["normed"]:
        out["normed"] = r.normed
    return out


def _own_quant(s):
    from lightop_amd.moe import act_and_mul_group_quant_fp8
    from lightop_amd.quant import per_token_group_quant_fp8

    act = s["case"]["activation"]
    q, scale = per_token_group_quant_fp8(s["x"], G) if act == "none" else act_and_mul_group_quant_fp8(s["x"], act)
    return {"q": q, "scale": scale}


def _own_gemm(s):
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    return {"out": gemm_w8a8_fp8_block(s["a"], s["b"], s["a_scale"], s["b_scale"], out_dtype=DTYPES[s["case"]["dtype"]])}


def _own_experts(s):
    from lightop_amd.moe import fused_experts_decode_fp8

    return {"out": fused_experts_decode_fp8(s["x"], s["w1"], s["w2"], s["weights"], s["ids"], s["w1_scale"], s["w2_scale"],
                                            activation=s["case"]["activation"], global_num_experts=LAYERS[s["case"]["layer"]][1],
                                            expert_map=s["map"], routed_scaling_factor=s["factor"], shared_output=s["shared"])}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "quant": _own_quant, "gemm": _own_gemm, "experts": _own_experts}[op](state)
    return {"norm": _plain_norm, "quant": _plain_quant, "gemm": _plain_gemm, "experts": _plain_experts}[op](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def _e4m3(v):
    """float64 values rounded to the nearest e4m3 value, ties to even: steps of 2^(e-3), 2^-9 below the normal ones."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    e = torch.where(torch.ldexp(torch.ones_like(v), e) > v.abs().clamp(min=2.0 ** -6), e - 1, e)
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _exact_groups(y):
    v = y.reshape(*y.shape[:-1], y.shape[-1] // G, G)
    amax = torch.maximum(v.abs().max(-1).values, torch.tensor(1e-10, dtype=torch.float64, device=y.device))
    return _e4m3(448.0 * v / amax[..., None]).reshape(y.shape), amax / 448.0


def _exact_act(name, h):
    g, u = h[..., :h.shape[-1] // 2], h[..., h.shape[-1] // 2:]
    return u * (g * torch.sigmoid(g) if name == "silu" else g * 0.5 * torch.erfc(-g / math.sqrt(2.0)))


def _exact_product(a, sa, b, sb):
    """a [m, k], b [n, k] codes as float64, one scale for 128 of a row's values and for 128 x 128 of b's."""
    sa = torch.kron(sa.double(), torch.ones(1, G, dtype=torch.float64, device=a.device))
    sb = torch.kron(sb.double(), torch.ones(G, G, dtype=torch.float64, device=a.device))[:b.shape[0]]
    return (a * sa) @ (b * sb).T


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double() + (0.0 if s["residual"] is None else s["residual"].double())
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * s["weight"].double()
        out = {} if s["residual"] is None else {"residual": x}
        if case["normed"]:
            out["normed"] = y
        if case["form"] == "fp8 groups":
            out["q"], out["scale"] = _exact_groups(y)
            return out
        rows = case["form"] == "int8 rows"
        v = y[:, None, :] if rows else y.reshape(y.shape[0], -1, G)
        scale = v.abs().max(-1, keepdim=True).values.clamp(min=1e-10) / 127.0
        q = (torch.round if rows else torch.trunc)(v / scale)
        if not rows:  # a group's maximum is its scale's 127-fold: the quotient of the two in 64 bits may fall a step short
            q = torch.trunc(v / scale * (1.0 + 2.0 ** -50))
        return {**out, "q": q.reshape(y.shape), "scale": scale.reshape(y.shape[0], -1)}
    if case["op"] == "quant":
        x = s["x"].double()
        q, scale = _exact_groups(x if case["activation"] == "none" else _exact_act(case["activation"], x))
        return {"q": q, "scale": scale}
    if case["op"] == "gemm":
        return {"out": _exact_product(s["a"].double(), s["a_scale"], s["b"].double(), s["b_scale"])}
    q, scale = _exact_groups(s["x"].double())
    out = torch.zeros(s["x"].shape, dtype=torch.float64, device=q.device)
    ids = s["ids"] if s["map"] is None else s["map"][s["ids"].long()]
    for e in sorted(set(ids.flatten().tolist()) - {-1}):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        h = _exact_product(q[t], scale[t], s["w1"][e].double(), s["w1_scale"][e])
        q2, scale2 = _exact_groups(_exact_act(case["activation"], h))
        y = _exact_product(q2, scale2, s["w2"][e].double(), s["w2_scale"][e])
        out.index_add_(0, t, y * s["weights"][t, j].double()[:, None])
    return {"out": out * s["factor"] + (0.0 if s["shared"] is None else s["shared"].double())}


def work(case):
    """Inputs once, outputs once; the products, and a handful of operations a value elsewhere."""
    M, b = int(case["tokens"]), BYTES[case["dtype"]]
    if case["op"] == "norm":
        H = case["hidden"]
        scales = M if case["form"] == "int8 rows" else M * H // G
        values = 1 + 2 * case["residual"] + case["normed"]
        return {"bytes": M * H * (values * b + 1) + H * b + 4 * scales, "flops": 10.0 * M * H}
    if case["op"] == "quant":
        C, gated = case["cols"], case["activation"] != "none"
        return {"bytes": M * C * (b * (2 if gated else 1) + 1) + 4 * M * C // G, "flops": (12.0 if gated else 3.0) * M * C}
    if case["op"] == "gemm":
        N, K = case["n"], case["k"]
        return {"bytes": M * K + N * K + 4 * (M + -(-N // G)) * (K // G) + M * N * b, "flops": 2.0 * M * N * K}
    E, Eg, k, H, I = LAYERS[case["layer"]]
    hit = E * (1.0 - (1.0 - k / Eg) ** M)
    rows = 3 if case["shared"] else 2
    return {"bytes": hit * 3 * I * H * (1 + 4 / (G * G)) + rows * M * H * b + 8 * M * k, "flops": 6.0 * M * k * E / Eg * I * H}
