"""The operators of a served layer's dense blocks, as cases to measure.

Five operators: the dense product of 16-bit operands with bias, activation and residual in its epilogue
(``gemm_bias_act``), both projections of a gated block with activation and product in one
(``gemm_act_and_mul``), the two of int8 rows and weights with a scale for each token and each weight row
(``gemm_w8a8_bias_act``, ``gemm_w8a8_act_and_mul``), and the norms behind and in front of a block with its gate
and residual scale (``rms_norm_block``).  Hidden and intermediate sizes are those of
``lightop_amd.workloads``; token counts run from one (a sequence decoding) to a prefill batch of 8192.

int8 codes come back as float32, which holds them exactly, times their scales: the values they stand for.
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
EPS = 1e-6

MAX_TOKENS = 8192
MAX_PRODUCT = 8192 * 4096 * 7168


def _gemm(tokens, n, k, dtype, weights="16", gated=False, activation="none", bias=False, residual=False, out=None):
    """``n``: columns of the result; a gated product has twice as many weight rows.  ``dtype`` is that of the rows, of
    the result where ``out`` does not say otherwise."""
    return {"op": "gemm", "tokens": tokens, "n": n, "k": k, "dtype": dtype, "weights": weights, "gated": gated, "activation": activation,
            "bias": bias, "residual": residual, "out": out or dtype}


def _norm(tokens, hidden, dtype, form, post, gate, sigmoid=False, normed=False, scales=False):
    return {"op": "norm", "tokens": tokens, "hidden": hidden, "dtype": dtype, "form": form, "post": post, "gate": gate, "sigmoid": sigmoid,
            "normed": normed, "scales": scales}


def listed():
    return [
        # router logits of one sequence decoding, fp32 as the top-k takes them
        dict(_gemm(1, 256, 7168, "bf16", out="fp32"), name="gemm, router 1"),
        # the down product of a decode batch, the residual added
        dict(_gemm(48, 7168, 2048, "bf16", residual=True), name="gemm, down 48"),
        # a narrow projection with a bias of a short chunk, no side a multiple of a tile
        dict(_gemm(333, 577, 7168, "fp16", bias=True), name="gemm, narrow 333"),
        # a projection of the largest prefill batch
        dict(_gemm(8192, 4096, 7168, "bf16", bias=True, residual=True), name="gemm, prefill 8192"),
        # first half of an unquantised shared expert, one sequence decoding
        dict(_gemm(1, 2048, 7168, "bf16", gated=True, activation="silu"), name="gated, decode 1"),
        # the same of a chunk of prefill with decode tokens riding along, GELU
        dict(_gemm(1531, 768, 2048, "fp16", gated=True, activation="gelu"), name="gated, chunk 1531"),
        # the int8 down product of a decode batch, the residual added
        dict(_gemm(24, 7168, 2048, "bf16", weights="int8", bias=True, residual=True), name="w8a8, down 24"),
        # an int8 projection of a prefill batch
        dict(_gemm(4096, 4096, 7168, "bf16", weights="int8"), name="w8a8, prefill 4096"),
        # first half of an int8 shared expert: one sequence decoding, a prefill batch
        dict(_gemm(1, 2048, 7168, "bf16", weights="int8", gated=True, activation="silu"), name="w8a8 gated, decode 1"),
        dict(_gemm(2003, 1536, 4096, "bf16", weights="int8", gated=True, activation="silu"), name="w8a8 gated, chunk 2003"),
        # one sequence decoding: the shared expert's gate, a scalar of the token, in front of int8 experts
        dict(_norm(1, 2048, "bf16", "int8 rows", True, "token", sigmoid=True), name="norm, int8 rows 1"),
        # the largest prefill batch: norms on both sides of a block, a channel's gate
        dict(_norm(8192, 7168, "bf16", "none", True, "channel", normed=True, scales=True), name="norm, both sides 8192"),
    ]


def draw(rng):
    def tokens(most):
        return min(most, max(1, round(math.exp(rng.uniform(0.0, math.log(most + 1))))))

    if rng.random() < 0.3:
        hidden = rng.choice((1024, 2048, 4096, 7168, G * rng.randint(1, 56)))
        form = rng.choice(("none", "int8 rows", "int8 groups", "fp8 groups"))
        gate = rng.choice(("none", "token", "channel", "full"))
        return _norm(tokens(MAX_TOKENS), hidden, rng.choice(("bf16", "bf16", "fp16", "fp32")), form, rng.random() < 0.7, gate,
                     sigmoid=gate != "none" and rng.random() < 0.5, normed=form == "none" or rng.random() < 0.3, scales=rng.random() < 0.5)
    gated, weights = rng.random() < 0.4, rng.choice(("16", "int8"))
    n, k = rng.choice(((4096, 7168), (7168, 2048), (1536, 2048), (768, 2048), (256, 7168), (128, 2048),
                       (rng.randint(1, 7168), 16 * rng.randint(1, 448))))
    if gated:
        n = (n + 1) // 2
    most = max(1, min(MAX_TOKENS, MAX_PRODUCT // (n * k * (2 if gated else 1))))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp16"))
    act = rng.choice(("silu", "silu", "gelu")) if gated else rng.choice(("none", "none", "silu", "gelu"))
    return _gemm(tokens(most), n, k, dtype, weights, gated, act, rng.random() < 0.4, not gated and rng.random() < 0.5,
                 rng.choice((dtype, dtype, dtype, "fp32")))


def _rows(g, rows, cols, dtype):
    """Activations: unit normal, one channel in 64 eight times as wide, as hidden states have them."""
    x = torch.randn(rows, cols, generator=g, dtype=torch.float32, device=g.device)
    x[:, ::64] *= 8.0
    return x.to(dtype)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, dtype=torch.float32, device=g.device)


def prepare(case, seed):
    dev, M = torch.device("cuda:0"), int(case["tokens"])
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + M)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "norm":
        H = case["hidden"]
        s["x"] = _rows(g, M, H, dtype)
        s["residual"] = (4.0 * _rows(g, M, H, torch.float32)).to(dtype)
        s["weight"] = (1.0 + 0.2 * _normal(g, H)).to(dtype)
        s["post"] = (1.0 + 0.2 * _normal(g, H)).to(dtype) if case["post"] else None
        shape = {"none": None, "token": (M, 1), "channel": (H,), "full": (M, H)}[case["gate"]]
        s["gate"] = None if shape is None else _normal(g, *shape).to(dtype)
        s["scale"], s["residual_scale"] = (0.22, 0.9) if case["scales"] else (1.0, 1.0)
        return s
    K, out = case["k"], DTYPES[case["out"]]
    N = case["n"] * (2 if case["gated"] else 1)
    if case["weights"] == "int8":
        rows = _rows(g, M, K, torch.float32)
        s["a_scale"] = rows.abs().amax(-1, keepdim=True) / 127.0
        s["a"] = torch.round(rows / s["a_scale"]).to(torch.int8)
        s["b"] = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8, device=dev)
        s["b_scale"] = torch.exp(0.3 * _normal(g, N, 1)) / (127.0 * math.sqrt(K))
    else:
        s["a"] = _rows(g, M, K, dtype)
        s["b"] = (_normal(g, N, K) / math.sqrt(K)).to(dtype)
    s["bias"] = _normal(g, N).to(out) if case["bias"] else None
    s["residual"] = (2.0 * _rows(g, M, case["n"], torch.float32)).to(out) if case["residual"] else None
    return s


# ---- the plain forms: torch.float32 between the inputs and one rounding of each output ----------------------------

def _activate(name, v):
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5))) if name == "gelu" else v


def _plain_gemm(s):
    c = s["case"]
    v = torch.matmul(s["a"].float(), s["b"].float().t())
    if c["weights"] == "int8":
        v = v * s["a_scale"] * s["b_scale"].view(-1)
    if s["bias"] is not None:
        v = v + s["bias"].float()
    if c["gated"]:
        v = _activate(c["activation"], v[:, :c["n"]]) * v[:, c["n"]:]
    else:
        v = _activate(c["activation"], v)
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return {"out": v.to(DTYPES[c["out"]])}


def _plain_norm(s):
    c, dtype = s["case"], s["x"].dtype
    h = s["x"].float()
    if c["post"]:
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["post"].float()
    if s["gate"] is not None:
        gate = s["gate"].float()
        h = h * (1.0 / (1.0 + torch.exp(-gate)) if c["sigmoid"] else gate)
    z = s["residual_scale"] * s["residual"].float() + s["scale"] * h
    y = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    out = {"residual": z.to(dtype)}
    if c["normed"]:
        out["normed"] = y.to(dtype)
    if c["form"] == "none":
        return out
    v = y.unsqueeze(-2) if c["form"] == "int8 rows" else y.unflatten(-1, (-1, G))
    amax = v.abs().amax(-1, keepdim=True).clamp(min=1e-10)
    if c["form"] == "fp8 groups":
        out["scale"] = (amax / 448.0).squeeze(-1)
        q = (v * 0.875 / (amax / 512.0)).to(FP8).float()
    else:
        out["scale"] = (amax / 127.0).squeeze(-1)
        q = torch.round(v * (127.0 / amax)) if c["form"] == "int8 rows" else torch.trunc(v / (amax / 127.0))
        q = q.clamp(-128, 127)
    out["values"] = (q * out["scale"].unsqueeze(-1)).flatten(-2)
    return out


# ---- the package's calls --------------------------------------------------------------------------------------------

def _own_gemm(s):
    from lightop_amd import gemmopt

    c, out = s["case"], DTYPES[s["case"]["out"]]
    act = None if c["activation"] == "none" else c["activation"]
    if c["weights"] == "int8":
        if c["gated"]:
            return {"out": gemmopt.gemm_w8a8_act_and_mul(s["a"], s["b"], s["a_scale"], s["b_scale"], bias=s["bias"], activation=act, out_dtype=out)}
        return {"out": gemmopt.gemm_w8a8_bias_act(s["a"], s["b"], s["a_scale"], s["b_scale"], bias=s["bias"], activation=act,
                                                  residual=s["residual"], out_dtype=out)}
    if c["gated"]:
        return {"out": gemmopt.gemm_act_and_mul(s["a"], s["b"], bias=s["bias"], activation=act, out_dtype=out)}
    return {"out": gemmopt.gemm_bias_act(s["a"], s["b"], bias=s["bias"], activation=act, residual=s["residual"], out_dtype=out)}


def _own_norm(s):
    from lightop_amd.norm import rms_norm_block

    c = s["case"]
    quant = {"none": (None, None), "int8 rows": (torch.int8, None), "int8 groups": (torch.int8, G), "fp8 groups": (FP8, G)}[c["form"]]
    r = rms_norm_block(s["x"], s["residual"], s["weight"], post_weight=s["post"], gate=s["gate"],
                       gate_activation="sigmoid" if c["sigmoid"] else None, scale=s["scale"], residual_scale=s["residual_scale"], eps=EPS,
                       quant_dtype=quant[0], group_size=quant[1], return_normed=c["normed"])
    out = {"residual": r.residual}
    if c["normed"]:
        out["normed"] = r.normed
    if c["form"] != "none":
        out["scale"] = r.scale
        q = r.q if r.q.dtype == torch.int8 else r.q.float()
        out["values"] = (q.unflatten(-1, (r.scale.shape[-1], -1)) * r.scale.unsqueeze(-1)).flatten(-2)
    return out


def run(state):
    if own:
        return {"gemm": _own_gemm, "norm": _own_norm}[state["case"]["op"]](state)
    return {"gemm": _plain_gemm, "norm": _plain_norm}[state["case"]["op"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def _e4m3(v):
    """float64 values rounded to the nearest e4m3 value, ties to even: steps of 2^(e-3), 2^-9 below the normal ones."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    e = torch.where(torch.ldexp(torch.ones_like(v), e) > v.abs().clamp(min=2.0 ** -6), e - 1, e)
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _exact_act(name, v):
    if name == "none":
        return v
    return v * torch.sigmoid(v) if name == "silu" else v * 0.5 * torch.erfc(-v / math.sqrt(2.0))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gemm":
        a, b = s["a"].double(), s["b"].double()
        if case["weights"] == "int8":
            a, b = a * s["a_scale"].double(), b * s["b_scale"].double()
        out = a @ b.T
        if s["bias"] is not None:
            out += s["bias"].double()
        if case["gated"]:
            gate, up = torch.tensor_split(out, 2, dim=1)
            out = _exact_act(case["activation"], gate) * up
        else:
            out = _exact_act(case["activation"], out)
        return {"out": out if s["residual"] is None else out + s["residual"].double()}
    x = s["x"].double()
    if case["post"]:
        x = s["post"].double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
    if case["gate"] != "none":
        gate = s["gate"].double()
        x = x * (torch.sigmoid(gate) if case["sigmoid"] else gate)
    z = s["residual"].double() * s["residual_scale"] + x * s["scale"]
    y = s["weight"].double() * z / torch.sqrt((z * z).sum(-1, keepdim=True) / z.shape[-1] + EPS)
    out = {"residual": z}
    if case["normed"]:
        out["normed"] = y
    if case["form"] == "none":
        return out
    v = y[:, None, :] if case["form"] == "int8 rows" else y.reshape(y.shape[0], -1, G)
    amax = v.abs().max(-1, keepdim=True).values.clamp(min=1e-10)
    most = 448.0 if case["form"] == "fp8 groups" else 127.0
    if case["form"] == "fp8 groups":
        q = _e4m3(v / amax * most)
    elif case["form"] == "int8 rows":
        q = torch.round(v / amax * most)
    else:  # a group's maximum is its scale's 127-fold: the quotient of the two in 64 bits may fall a step short
        q = torch.trunc(v / amax * most * (1.0 + 2.0 ** -50))
    out["scale"] = (amax / most).reshape(y.shape[0], -1)
    out["values"] = (q * amax / most).reshape(y.shape)
    return out


def work(case):
    """Inputs once, outputs once; the products, and a handful of operations a value elsewhere."""
    M, b = int(case["tokens"]), BYTES[case["dtype"]]
    if case["op"] == "norm":
        H = case["hidden"]
        gate = {"none": 0, "token": M, "channel": H, "full": M * H}[case["gate"]]
        code = 0 if case["form"] == "none" else 1
        scales = 0 if case["form"] == "none" else M if case["form"] == "int8 rows" else M * H // G
        return {"bytes": M * H * (3 * b + case["normed"] * b + code) + gate * b + (2 if case["post"] else 1) * H * b + 4 * scales,
                "flops": (16.0 if case["post"] else 11.0) * M * H}
    n, K, o = case["n"], case["k"], BYTES[case["out"]]
    N = n * (2 if case["gated"] else 1)
    size, scales = (1, 4 * (M + N)) if case["weights"] == "int8" else (b, 0)
    return {"bytes": (M + N) * K * size + scales + case["bias"] * N * o + M * n * o * (2 if case["residual"] else 1),
            "flops": 2.0 * M * N * K}
