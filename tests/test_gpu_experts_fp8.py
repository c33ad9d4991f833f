"""The experts of a few tokens with e4m3 weights against float64: the first product's activations out of the workspace, the output from them."""
import ctypes

import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu


def _layer(E, H, I, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + E + H + I)
    w1, s1 = ref.weights((E, 2 * I, H), g, "cuda")
    w2, s2 = ref.weights((E, H, I), g, "cuda")
    return w1, w2, s1, s2


def _tokens(M, H, Eg, k, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(100 + seed + M)
    x = ref.rows(M, H, g, "cuda", dtype)
    p, ids = torch.topk(torch.softmax(torch.randn(M, Eg, generator=g, device="cuda"), -1), k, dim=-1)
    return x, p / p.sum(-1, keepdim=True), ids.int(), ref.rows(M, H, g, "cuda", dtype)


def _local(ids, emap, E):
    """Local expert of every slot, -1 where there is none."""
    ids = ids.long()
    Eg = E if emap is None else emap.numel()
    inside = (ids >= 0) & (ids < Eg)
    e = ids.clamp(0, Eg - 1)
    e = e if emap is None else emap.long()[e]
    return torch.where(inside & (e >= 0) & (e < E), e, -1)


def _run(x, w, tw, ids, emap=None, act="silu", factor=1.0, shared=None):
    """Through the C entry point: (out, the fp32 activations [M, k, I])."""
    from lightop_amd import _lib

    w1, w2, s1, s2 = w
    M, H = x.shape
    E, I, k = w1.shape[0], w1.shape[1] // 2, ids.shape[1]
    lib = _lib.lib()
    n = lib.lo_fused_experts_fp8_workspace_bytes(M, k, H, I)
    ws = torch.full((n,), 0xff, dtype=torch.uint8, device="cuda")  # NaN wherever nothing is written
    out = torch.empty_like(x)
    _lib.check(lib.lo_fused_experts_fp8(
        _lib.ptr(x), {torch.bfloat16: 0, torch.float16: 1}[x.dtype], M, H, I, E, E if emap is None else emap.numel(), k, _lib.ptr(w1),
        _lib.ptr(s1), _lib.ptr(w2), _lib.ptr(s2), _lib.ptr(tw), _lib.ptr(ids), 1 if ids.dtype == torch.int64 else 0, _lib.ptr(emap),
        1 if act == "gelu" else 0, factor, _lib.ptr(shared), _lib.ptr(out), _lib.ptr(ws), n, _lib.stream_of(x)))
    return out, ws[:M * k * I * 4].view(torch.float32).view(M, k, I)


def _codes32(v):
    """The rule on fp32 values, step by step as the kernel rounds it."""
    g = v.unflatten(-1, (-1, 128))
    top = g.abs().amax(-1).clamp(min=1e-10)
    return ref.e4m3(((g * 0.875) / (top / 512).unsqueeze(-1)).double()).flatten(-2), top / 448


def _check(x, w, tw, ids, emap=None, act="silu", factor=1.0, shared=None):
    w1, w2, s1, s2 = w
    out, h = _run(x, w, tw, ids, emap, act, factor, shared)
    E, k = w1.shape[0], ids.shape[1]
    e = _local(ids, emap, E)
    q, s = _codes32(x.float())
    xd = ref.dequant(q, s)
    want = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    slack = torch.zeros_like(want)
    KB1, KB2 = w1.shape[2] // 128, w2.shape[2] // 128
    for t in range(x.shape[0]):
        first = {}
        for j in range(k):
            n = int(e[t, j])
            if n < 0:
                continue
            if n not in first:
                first[n] = j
                d1 = ref.dequant_weight(w1[n], s1[n])
                g = xd[t] @ d1.T
                # fp32 sums of exact products: a rounding a step of K and of a product's 128 values; the activation multiplies either half
                off = (xd[t].abs() @ d1.abs().T) * (KB1 + 140) * ref.ULP32
                v = ref.act_mul(act, g)
                I = v.numel()
                # |d act / dg| is at most 1.13
                tol = 1.13 * off[:I] * (g[I:].abs() + off[I:]) + off[I:] * g[:I].abs() + v.abs() * 2.0 ** -20
                if act == "gelu":
                    tol = tol + v.abs() * g[:I].square() * ref.ULP32
                assert ((h[t, j].double() - v).abs() <= tol + 1e-30).all(), (t, j)
            hq, hs = _codes32(h[t, first[n]])
            d2 = ref.dequant_weight(w2[n], s2[n])
            hd = ref.dequant(hq, hs)
            y = float(tw[t, j]) * (hd @ d2.T)
            want[t] += y
            # fp32 sums, and what an e4m3 instruction drops: at most 2^-11 of a K block's largest product
            tops = lambda m: m.abs().unflatten(-1, (-1, 128)).amax(-1)
            slack[t] += float(tw[t, j]) * ((hd.abs() @ d2.abs().T) * (KB2 + 150 + k) * ref.ULP32 + 2.0 ** -11 * (tops(hd) @ tops(d2).T))
    want, slack = want * factor, slack * abs(factor)
    if shared is not None:
        want = want + shared.double()
    assert ((out.double() - want).abs() <= slack + 1.01 * ref.half_step(x.dtype, want) + 4 * ref.ULP32 * want.abs()).all()
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M", [1, 2, 5, 16, 17, 33, 64])
@pytest.mark.parametrize("E,k,H,I", [(8, 2, 1024, 512), (3, 1, 128, 128), (40, 6, 384, 896), (1, 1, 256, 128)])
def test_values(dtype, act, M, E, k, H, I):
    print("[case] experts", dtype, act, M, E, k, H, I, flush=True)
    x, tw, ids, shared = _tokens(M, H, E, k, dtype)
    _check(x, _layer(E, H, I), tw, ids, act=act, shared=shared if M % 2 else None, factor=2.5 if M % 2 else 1.0)


@pytest.mark.parametrize("M", [1, 3, 20, 64])
def test_share_of_the_experts(M):
    """A map that leaves tokens without any expert here, ids out of range, int64 ids."""
    w = _layer(4, 512, 256)
    x, tw, ids, shared = _tokens(M, 512, 16, 4, torch.bfloat16)
    emap = torch.full((16,), -1, dtype=torch.int32, device="cuda")
    emap[[2, 5, 6, 11]] = torch.tensor([3, 0, 2, 1], dtype=torch.int32, device="cuda")
    ids[0] = torch.tensor([0, 1, 3, 4], dtype=torch.int32, device="cuda")  # none here
    out = _check(x, w, tw, ids, emap, shared=shared)
    assert torch.equal(out[0], shared[0])
    assert (_run(x, w, tw, ids, emap)[0][0] == 0).all()
    ids[M - 1] = torch.tensor([-1, 16, 2, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    _check(x, w, tw, ids, emap)
    a = _run(x, w, tw, ids.long(), emap)[0]
    assert torch.equal(a, _run(x, w, tw, ids, emap)[0])
    emap[5] = 77  # an entry outside of the weights
    _check(x, w, tw, ids, emap)
    nobody = torch.full_like(emap, -1)
    assert (_run(x, w, tw, ids, nobody)[0] == 0).all()


@pytest.mark.parametrize("M,E", [(2, 64), (9, 6), (64, 2)])
def test_an_expert_twice_in_a_token(M, E):
    w = _layer(E, 256, 128)
    x, tw, ids, _ = _tokens(M, 256, E, 2, torch.float16)
    ids = torch.cat([ids, ids.flip(1), ids[:, :1]], dim=1).contiguous()
    tw = torch.rand(M, 5, device="cuda")
    _check(x, w, tw, ids)


@pytest.mark.parametrize("M", [17, 64])
def test_every_token_on_one_expert(M):
    w = _layer(32, 512, 256)
    x, tw, ids, _ = _tokens(M, 512, 32, 2, torch.bfloat16)
    ids[:, 0] = 31
    ids[:, 1] = torch.arange(M, device="cuda") % 31
    _check(x, w, tw, ids)


def test_widest_call():
    w = _layer(128, 128, 128)
    x, tw, ids, _ = _tokens(64, 128, 128, 16, torch.bfloat16)
    _check(x, w, tw, ids)


def test_entry_point(monkeypatch):
    from lightop_amd import _lib
    from lightop_amd.moe import fused_experts_decode_fp8

    w1, w2, s1, s2 = w = _layer(8, 1024, 512)
    x, tw, ids, shared = _tokens(5, 1024, 8, 2, torch.bfloat16)
    want = _run(x, w, tw, ids, factor=1.5, shared=shared)[0]
    call = lambda x, tw=tw, ids=ids, **k: fused_experts_decode_fp8(x, w1, w2, tw, ids, s1, s2, routed_scaling_factor=1.5,
                                                                  shared_output=shared, **k)
    assert torch.equal(call(x), want)
    with monkeypatch.context() as m:
        m.setattr(_lib, "_host", _lib._NoHost())
        assert torch.equal(call(x), want)
    y = x.clone()
    assert call(y, inplace=True).data_ptr() == y.data_ptr() and torch.equal(y, want)
    assert torch.equal(call(x.t().contiguous().t(), tw.t().contiguous().t(), ids.t().contiguous().t()), want)
    assert torch.equal(call(torch.cat([x, x], 1)[:, :1024]), want)
    off = torch.zeros(5 * 1024 + 1, dtype=x.dtype, device="cuda")[1:].view(5, 1024).copy_(x)
    assert torch.equal(call(off), want)
    assert fused_experts_decode_fp8(x[:0], w1, w2, tw[:0], ids[:0], s1, s2).shape == (0, 1024)
    f = fused_experts_decode_fp8
    big = torch.zeros(65, 1024, dtype=torch.bfloat16, device="cuda")
    for bad, kind in ((lambda: f(big, w1, w2, torch.ones(65, 2, device="cuda"), torch.zeros(65, 2, dtype=torch.int32, device="cuda"), s1, s2),
                       RuntimeError), (lambda: f(x.float(), w1, w2, tw, ids, s1, s2), NotImplementedError),
                      (lambda: f(x, w1.float(), w2, tw, ids, s1, s2), RuntimeError), (lambda: f(x, w1, w2, tw, ids.float(), s1, s2), RuntimeError),
                      (lambda: f(x, w1, w2[:4], tw, ids, s1, s2), AssertionError), (lambda: f(x, w1, w2, tw[:4], ids, s1, s2), AssertionError),
                      (lambda: f(x, w1, w2, tw, ids, s1[:, :4], s2), AssertionError), (lambda: f(x, w1, w2, tw, ids, s1, s2, "relu"), ValueError),
                      (lambda: f(x, w1, w2, tw, ids, s1, s2, global_num_experts=16), RuntimeError),
                      (lambda: f(x, w1, w2, tw, ids, s1, s2.cpu()), RuntimeError),
                      (lambda: f(x, w1, w2, tw, ids, s1, s2, global_num_experts=16, expert_map=ids[0]), RuntimeError),
                      (lambda: f(x, w1, w2, tw, ids, s1, s2, shared_output=x[:2]), RuntimeError)):
        with pytest.raises(kind):
            bad()


def test_streams_and_graphs():
    """Two graphs and eager calls on two streams keep out of each other's scratch."""
    from lightop_amd.moe import fused_experts_decode_fp8

    w1, w2, s1, s2 = _layer(8, 1024, 512)
    sets = [_tokens(9, 1024, 8, 2, torch.bfloat16, seed=i) for i in range(3)]
    f = lambda x, tw, ids, sh: fused_experts_decode_fp8(x, w1, w2, tw, ids, s1, s2, shared_output=sh)
    want = [f(*s) for s in sets]
    graphs = []
    for i in range(2):
        hold = [t.clone() for t in sets[i]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f(*hold)
        graphs.append((graph, hold, out))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for r in range(4):
        for i, (graph, hold, out) in enumerate(graphs):
            for h, t in zip(hold, sets[(r + i) % 3]):
                h.copy_(t)
            graph.replay()
        with torch.cuda.stream(side):
            other = f(*sets[r % 3])
        here = f(*sets[(r + 1) % 3])
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][2], want[r % 3]) and torch.equal(graphs[1][2], want[(r + 1) % 3])
        assert torch.equal(other, want[r % 3]) and torch.equal(here, want[(r + 1) % 3])


@pytest.mark.parametrize("M,k,E", [(16, 64, 2048), (1, 64, 64), (1, 64, 2048), (64, 1, 2048), (64, 16, 2048), (13, 2, 24), (12, 2, 25), (64, 1, 1)])
def test_limits(M, k, E):
    """The most tokens, slots, slots a token and experts, and both sides of the step from two launches to four."""
    print("[case] experts", M, k, E, flush=True)
    w = _layer(E, 128, 128)
    x, tw, ids, shared = _tokens(M, 128, E, k, torch.bfloat16)
    _check(x, w, tw, ids, shared=shared)


@pytest.mark.parametrize("M,E,k,H,I", [(16, 26, 4, 4096, 256), (64, 26, 3, 4224, 128), (30, 30, 6, 2048, 1152), (64, 8, 16, 256, 1024)])
def test_widths_of_many_experts_hit(M, E, k, H, I):
    """Column blocks of one workgroup (4096 columns up) and of two; parts of K of unequal lengths, and as many as the sums' room allows."""
    print("[case] experts", M, E, k, H, I, flush=True)
    w = _layer(E, H, I)
    x, tw, ids, shared = _tokens(M, H, E, min(k, E), torch.float16)
    if k > E:
        ids, tw = ids.repeat(1, 2)[:, :k].contiguous(), tw.repeat(1, 2)[:, :k].contiguous()
    a = _check(x, w, tw, ids, shared=shared, factor=0.5)
    for _ in range(4):  # the same bits every time
        assert torch.equal(_run(x, w, tw, ids, shared=shared, factor=0.5)[0], a)


@pytest.mark.parametrize("M", [3, 48])
def test_nans_and_infinities_stay_where_they_are(M):
    w = _layer(32, 512, 256)
    x, tw, ids, shared = _tokens(M, 512, 32, 4, torch.bfloat16)
    want = _run(x, w, tw, ids, shared=shared)[0]
    bad, bw, bi = x.clone(), tw.clone(), ids.clone()
    bad[1, 7], bad[2, 300] = float("nan"), float("inf")
    out = _run(bad, w, tw, ids, shared=shared)[0]
    keep = [t for t in range(M) if t not in (1, 2)]
    assert torch.equal(out[keep], want[keep]) and not out[1].isfinite().any() and not out[2].isfinite().any()
    bi[:, 3], bw[:, 3] = -1, 0.0
    none = _run(x, w, bw, bi, shared=shared)[0]
    for v in (float("nan"), float("inf")):  # weights of slots without an expert are not looked at
        bw[:, 3] = v
        assert torch.equal(_run(x, w, bw, bi, shared=shared)[0], none)


@pytest.mark.parametrize("M,H", [(40, 1024), (20, 4096)])
def test_streams_graphs_and_threads_of_many_slots(M, H):
    """Two captured graphs, a thread on a stream of its own, another one on this one's stream: each with its own scratch, or in turn."""
    import threading

    from lightop_amd.moe import fused_experts_decode_fp8

    w1, w2, s1, s2 = _layer(24, H, 256)
    sets = [_tokens(M, H, 24, 4, torch.bfloat16, seed=i) for i in range(3)]
    f = lambda x, tw, ids, sh: fused_experts_decode_fp8(x, w1, w2, tw, ids, s1, s2, shared_output=sh)
    want = [f(*s) for s in sets]
    graphs = []
    for i in range(2):
        hold = [t.clone() for t in sets[i]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f(*hold)
        graphs.append((graph, hold, out))
    torch.cuda.synchronize()
    main, made = torch.cuda.current_stream(), {}

    def work(name, stream):
        with torch.cuda.stream(stream):
            made[name] = [f(*sets[i % 3]) for i in range(30)]
            stream.synchronize()

    for r in range(3):
        threads = [threading.Thread(target=work, args=("own", torch.cuda.Stream())), threading.Thread(target=work, args=("same", main))]
        for t in threads:
            t.start()
        for i, (graph, hold, out) in enumerate(graphs):
            for h, t in zip(hold, sets[(r + i) % 3]):
                h.copy_(t)
            graph.replay()
        here = [f(*sets[i % 3]) for i in range(30)]
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][2], want[r % 3]) and torch.equal(graphs[1][2], want[(r + 1) % 3])
        for outs in (made["own"], made["same"], here):
            assert all(torch.equal(o, want[i % 3]) for i, o in enumerate(outs))


@pytest.mark.parametrize("M,k", [(8192, 2), (64, 20), (1, 65)])
def test_a_refused_batch_takes_no_memory(monkeypatch, M, k):
    """More tokens or slots than a call takes: refused before a workspace of that size is made, or kept."""
    from lightop_amd import _lib
    from lightop_amd.moe import fused_experts_decode_fp8

    w1, w2, s1, s2 = _layer(4, 256, 512)
    x = torch.zeros(M, 256, dtype=torch.bfloat16, device="cuda")
    tw, ids = torch.ones(M, k, device="cuda"), torch.zeros(M, k, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()  # (its own workspace, none so far)

    def refused():
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        with torch.cuda.stream(side), pytest.raises(RuntimeError, match="fused_experts_fp8"):
            fused_experts_decode_fp8(x, w1, w2, tw, ids, s1, s2)
        assert torch.cuda.memory_allocated() == before and torch.cuda.max_memory_allocated() == before

    refused()
    monkeypatch.setattr(_lib, "_host", _lib._NoHost())
    refused()


@pytest.mark.parametrize("M,E,k", [(5, 8, 2), (40, 32, 4)])
def test_in_place_beside_shared_rows(M, E, k):
    """The output over the hidden states, which are the shared rows too, or follow them in one buffer; shifted by a row it is refused."""
    from lightop_amd.moe import fused_experts_decode_fp8

    w1, w2, s1, s2 = _layer(E, 256, 128)
    x, tw, ids, shared = _tokens(M, 256, E, k, torch.bfloat16)
    f = lambda x, sh, **o: fused_experts_decode_fp8(x, w1, w2, tw, ids, s1, s2, shared_output=sh, **o)
    want, own = f(x, shared), f(x, x)
    y = x.clone()
    assert torch.equal(f(y, y, inplace=True), own) and torch.equal(y, own)
    buf = torch.cat([shared, x])
    assert torch.equal(f(buf[M:], buf[:M], inplace=True), want)
    assert torch.equal(buf[M:], want) and torch.equal(buf[:M], shared)
    buf = torch.cat([x, x])
    with pytest.raises(RuntimeError, match="overlaps"):
        f(buf[1:M + 1], buf[:M], inplace=True)
    assert torch.equal(buf, torch.cat([x, x]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M,E,k,H,I", [(32, 30, 4, 2048, 768), (16, 26, 8, 4096, 256)])
def test_many_experts_hit_only_fp32_roundings_are_in_front_of_the_output(dtype, M, E, k, H, I):
    """The second product of the four launches keeps its sums to fp32's precision."""
    w1, w2, s1, s2 = w = _layer(E, H, I)
    x, tw, ids, _ = _tokens(M, H, E, k, dtype)
    out, h = _run(x, w, tw, ids)
    want, slack = torch.zeros(M, H, dtype=torch.float64, device="cuda"), torch.zeros(M, H, dtype=torch.float64, device="cuda")
    for e in range(E):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if not t.numel():
            continue
        hd, d2, share = ref.dequant(*_codes32(h[t, j])), ref.dequant_weight(w2[e], s2[e]), tw[t, j].double().unsqueeze(1)
        want.index_add_(0, t, share * (hd @ d2.T))
        slack.index_add_(0, t, share * (hd.abs() @ d2.abs().T) * (I // 128 + 150 + k) * ref.ULP32)
    assert ((out.double() - want).abs() <= slack + ref.half_step(dtype, want.abs() + slack)).all()
