"""Dense products with bias, activation and residual, and both projections of a gated block, against float64."""
import pytest
import torch

import dense_ref as ref

pytestmark = pytest.mark.gpu

KINDS = [torch.bfloat16, torch.float16, torch.int8]
# bias ("out": of the result's type), activation, residual, scale, result's type (None: the default)
PLAIN = [(None, None, False, 1.0, None), ("out", None, True, 1.0, None), (torch.float32, "silu", False, 0.5, torch.float16),
         ("out", "gelu", True, 2.5, torch.float32), (None, None, False, 1.0, torch.float32), (None, "silu", True, -1.0, torch.bfloat16)]
GATED = [(None, "silu", None), ("out", "gelu", None), (torch.float32, "silu", torch.float32), (None, "gelu", torch.float16)]


def _out(kind, out):
    return out or (torch.bfloat16 if kind == torch.int8 else kind)


def _call(a, b, sa, sb, gated, **k):
    from lightop_amd import gemmopt

    if sa is None:
        return (gemmopt.gemm_act_and_mul if gated else gemmopt.gemm_bias_act)(a, b, **k)
    if k.get("out_dtype", 0) is None:
        del k["out_dtype"]
    return (gemmopt.gemm_w8a8_act_and_mul if gated else gemmopt.gemm_w8a8_bias_act)(a, b, sa, sb, **k)


def _case(kind, M, N, K, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + M * 7 + N * 3 + K)
    return g, ref.operands(kind, M, N, K, g)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("M", [1, 2, 4, 5, 15, 16, 17, 33, 48, 64, 65, 100, 128, 129, 200, 257, 400, 777])
@pytest.mark.parametrize("N,K", [(1, 16), (17, 400), (128, 1024), (576, 2048), (1001, 656), (2048, 784)])
def test_plain(kind, M, N, K):
    print("[case] dense", kind, M, N, K, flush=True)
    g, ops = _case(kind, M, N, K)
    for bias, activation, residual, scale, out in PLAIN:
        dtype = _out(kind, out)
        bias = None if bias is None else _normal(g, N).to(dtype if bias == "out" else bias)
        r = (2 * _normal(g, M, N)).to(dtype) if residual else None
        got = _call(*ops, False, bias=bias, activation=activation, residual=r, scale=scale, out_dtype=out)
        assert got.dtype == dtype
        ref.check(got, ref.dense(*ops, bias, activation, False, r, scale))


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("M", [1, 3, 4, 7, 16, 17, 48, 64, 65, 128, 190, 257, 600])
@pytest.mark.parametrize("N,K", [(1, 32), (9, 144), (64, 1024), (383, 848), (768, 2048), (1024, 272)])
def test_gated(kind, M, N, K):
    print("[case] gated", kind, M, N, K, flush=True)
    g, ops = _case(kind, M, 2 * N, K, 1)
    for bias, activation, out in GATED:
        dtype = _out(kind, out)
        bias = None if bias is None else _normal(g, 2 * N).to(dtype if bias == "out" else bias)
        ref.check(_call(*ops, True, bias=bias, activation=activation, out_dtype=out), ref.dense(*ops, bias, activation, True))


@pytest.mark.parametrize("K", [8, 24, 56, 64, 72, 120, 136, 504, 520])
@pytest.mark.parametrize("M", [3, 40, 130])
def test_k_of_sixteen_bits_in_eights(K, M):
    g, ops = _case(torch.bfloat16, M, 96, K)
    ref.check(_call(*ops, False), ref.dense(*ops))
    ref.check(_call(*ops, True), ref.dense(*ops, activation="silu", gated=True))


@pytest.mark.parametrize("kind,M,N,K,gated", [
    (torch.bfloat16, 1, 256, 7168, False), (torch.bfloat16, 48, 7168, 2048, False), (torch.float16, 333, 577, 7168, False),
    (torch.bfloat16, 4099, 4096, 1152, False), (torch.bfloat16, 1, 2048, 7168, True), (torch.float16, 1531, 768, 2048, True),
    (torch.int8, 24, 7168, 2048, False), (torch.int8, 2048, 2048, 2048, False), (torch.int8, 1, 2048, 7168, True),
    (torch.int8, 2003, 1536, 4096, True), (torch.int8, 5, 40, 131056, False), (torch.int8, 300, 264, 16384, False)])
def test_full_sizes(kind, M, N, K, gated):
    print("[case] dense", kind, M, N, K, gated, flush=True)
    g, ops = _case(kind, M, 2 * N if gated else N, K)
    k = dict(activation="silu" if gated else None)
    out = _call(*ops, gated, **k)
    ref.check(out, ref.dense(*ops, gated=gated, **k))
    assert torch.equal(out, _call(*ops, gated, **k))  # one order of the sum


@pytest.mark.parametrize("tile,size", ref.TILE_SIZES, ids=str)
def test_ragged_sizes_of_every_tile(tile, size):
    """Each tile, whole and in parts, plain and gated, every operand type, every way out of its epilogue."""
    M, N, K = size
    gated = tile[3]
    for kind, out, k in ((torch.bfloat16, None, K), (torch.float16, torch.float32, K), (torch.int8, torch.float16, 2 * K), (torch.int8, torch.float32, 2 * K)):
        print("[case] dense", tile, kind, M, N, k, flush=True)
        g, ops = _case(kind, M, 2 * N if gated else N, k, 2)
        dtype = _out(kind, out)
        more = dict(bias=_normal(g, 2 * N if gated else N).to(dtype), activation="silu" if gated else None)
        if not gated:
            more.update(residual=_normal(g, M, N).to(dtype), scale=0.75)
        ref.check(_call(*ops, gated, out_dtype=out, **more), ref.dense(*ops, gated=gated, **more))


@pytest.mark.parametrize("size", ref.FEW, ids=str)
def test_every_form_of_few_tokens(size):
    M, N, K, gated = size
    print("[case] few", *size, flush=True)
    for kind, k in ((torch.bfloat16, K), (torch.float16, K), (torch.int8, 2 * K)):
        g, ops = _case(kind, M, 2 * N if gated else N, k, 3)
        bias = _normal(g, 2 * N if gated else N)
        r = None if gated else _normal(g, M, N).to(_out(kind, None))
        got = _call(*ops, gated, bias=bias, activation="silu" if gated else None, **({} if gated else {"residual": r}))
        ref.check(got, ref.dense(*ops, bias, "silu" if gated else None, gated, r))


def test_int8_sums_are_exact():
    """All products of one sign and largest: K * 2^14, just under 2^31."""
    for M in (1, 20, 200):
        a = torch.full((M, 131056), -128, dtype=torch.int8, device="cuda")
        b = torch.full((40, 131056), -128, dtype=torch.int8, device="cuda")
        one = torch.ones(M, device="cuda"), torch.ones(40, device="cuda")
        out = _call(a, b, *one, False, out_dtype=torch.float32)
        assert (out == 131056 * 2.0 ** 14).all()


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [1, 3, 16, 40, 70, 300, 600])
@pytest.mark.parametrize("N", [40, 250, 520])
def test_nothing_else_is_written_or_read(kind, gated, M, N):
    """Rows of either operand that lie in a wider tensor full of NaNs (int8: of 127), K that ends inside a block; values
    around the result stay; a NaN stays in its row or column."""
    g, (a, b, sa, sb) = _case(kind, M, 2 * N if gated else N, 208)
    want = _call(a, b, sa, sb, gated)
    fill = 127 if kind == torch.int8 else float("nan")
    wide = [torch.full((t.shape[0] + 2, 288), fill, dtype=kind, device="cuda") for t in (a, b)]
    for w, t in zip(wide, (a, b)):
        w[1:-1, 32:240] = t
    room = torch.full((M * N + 4096,), 7.0, dtype=want.dtype, device="cuda")
    out = room[2048:2048 + M * N].view(M, N)
    got = _call(wide[0][1:-1, 32:240], wide[1][1:-1, 32:240], sa, sb, gated, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
    assert (room[:2048] == 7).all() and (room[2048 + M * N:] == 7).all()
    if kind == torch.int8:
        sa, sb = sa.clone(), sb.clone()
        sa[M - 1] = float("nan")
        sb[N - 1] = float("nan")
    else:
        a, b = a.clone(), b.clone()
        a[M - 1, 5] = float("nan")
        b[N - 1, 200] = float("nan")
    got = _call(a, b, sa, sb, gated)
    assert got[M - 1].isnan().all() and got[:, N - 1].isnan().all() and torch.equal(got[:-1, :-1], want[:-1, :-1])


@pytest.mark.parametrize("M", [2, 40, 300])
def test_infinities_and_far_values(M):
    """An infinity, the type's lowest values and gates far from zero give what the formula gives; nothing else changes."""
    for kind in (torch.bfloat16, torch.float16):
        g, (a, b, _, _) = _case(kind, M, 80, 128)
        a, b = torch.zeros_like(a), torch.zeros_like(b)
        a[:, 0] = 1.0
        gates = torch.tensor([float("inf"), -float("inf"), 1e4, -1e4, -200.0, -90.0, -30.0, -8.0, -1e-3, 0.0], device="cuda")
        b[:10, 0] = gates.to(kind)
        b[40:50, 0] = 1.0
        for name in ("silu", "gelu"):
            got = _call(a, b, None, None, True, activation=name, out_dtype=torch.float32)
            v = b[:10, 0].double()
            want = ref.act(name, v)
            assert got[0, 0] == float("inf") and got[0, 1].isnan()  # -inf * 0
            # gelu: erfc's argument z = |g| / sqrt 2 carries the constant's and the product's rounding, 2 * 2^-24 of it; far out erfc falls as
            # exp(-z^2), whose relative change 2 z dz is then 4 z^2 2^-24 = 2 g^2 2^-24
            rel = 1e-6 + (2 * v[2:] ** 2 * 2.0 ** -24 if name == "gelu" else 0.0)
            assert ((got[:, 2:10].double() - want[2:]).abs() <= rel * want[2:].abs() + 1e-37).all()
            assert (got[:, 10:] == 0).all()
        low = torch.finfo(kind).min
        a[:, 0], b[:, 0] = low, 1.0
        assert (_call(a, b, None, None, False) == low).all()
        assert (_call(a, b, None, None, False, scale=2.0) == -float("inf")).all()


def test_zero_rows_and_columns():
    for kind in KINDS:
        g, (a, b, sa, sb) = _case(kind, 70, 130, 256)
        cut = lambda t, n: None if t is None else t[:n]
        assert _call(a[:0], b, cut(sa, 0), sb, False).shape == (0, 130)
        assert _call(a, b[:0], sa, cut(sb, 0), False).shape == (70, 0)
        assert _call(a, b[:0], sa, cut(sb, 0), True).shape == (70, 0)
        bias = _normal(g, 130)
        r = _normal(g, 70, 130)
        out = _call(torch.zeros_like(a), b, sa, sb, False, bias=bias, residual=r, out_dtype=torch.float32)
        assert torch.equal(out, bias + r)


@pytest.mark.parametrize("kind,M,N,K,gated", [(torch.bfloat16, 160000, 24, 7168, False), (torch.bfloat16, 40, 160000, 7168, False),
                                              (torch.bfloat16, 40, 80000, 7168, True), (torch.float16, 70000, 16384, 128, False),
                                              (torch.int8, 2, 310000, 7168, False), (torch.int8, 310000, 24, 7168, False)])
def test_offsets_past_32_bits(kind, M, N, K, gated):
    """Operands and results of more than 2 GiB: the last rows and columns."""
    print("[case] dense", kind, M, N, K, gated, flush=True)
    g, (a, b, sa, sb) = _case(kind, M, 2 * N if gated else N, K)
    out = _call(a, b, sa, sb, gated)
    m, n = min(M, 200), min(N, 200)
    halves = ((0, n), (N - n, N))
    for lo, hi in halves:
        w = torch.cat([b[lo:hi], b[N + lo:N + hi]]) if gated else b[lo:hi]
        ws = None if sb is None else sb[lo:hi]
        for r in (slice(0, m), slice(M - m, M)):
            want = ref.dense(a[r], w, None if sa is None else sa[r], ws, activation="silu" if gated else None, gated=gated)
            ref.check(out[r, lo:hi], want)


def test_strides_batches_and_marshalling(monkeypatch):
    from lightop_amd import _lib

    for kind in KINDS:
        g, (a, b, sa, sb) = _case(kind, 24, 96, 256)
        bias, r = _normal(g, 96), _normal(g, 24, 96).to(_out(kind, None))
        k = dict(bias=bias, activation="gelu")
        want = _call(a, b, sa, sb, False, residual=r, **k)
        pair = lambda t: None if t is None else t.view(2, 12, -1)
        got = _call(pair(a), b, pair(sa), sb, False, residual=pair(r), **k)
        assert got.shape == (2, 12, 96) and torch.equal(got.view(24, 96), want)
        if sa is not None:
            assert torch.equal(_call(pair(a), b, sa.view(2, 12), sb.view(96, 1), False, residual=pair(r), **k), got)
        one = _call(a[3], b, None if sa is None else sa[3], sb, False, residual=r[3], **k)
        assert one.shape == (96,)
        ref.check(one[None], ref.dense(a[3:4], b, None if sa is None else sa[3:4], sb, bias, "gelu", False, r[3:4]))
        off = torch.zeros(24 * 256 + 1, dtype=kind, device="cuda")[1:].view(24, 256).copy_(a)
        turned = b.t().contiguous().t()
        every = r.repeat_interleave(2, 0)[::2]
        assert torch.equal(_call(off, turned, sa, sb, False, residual=every, **k), want)
        spread = torch.zeros(24, 192, dtype=r.dtype, device="cuda")[:, ::2].copy_(r)
        assert torch.equal(_call(a, b, sa, sb, False, residual=spread, **k), want)
        wide = torch.zeros(24, 101, dtype=r.dtype, device="cuda")[:, 3:99].copy_(r)  # rows that begin off 16 bytes
        assert torch.equal(_call(a, b, sa, sb, False, residual=wide, **k), want)
        same = _call(a[:1].expand(24, 256), b, None if sa is None else sa[:1].expand(24, 1), sb, False)
        assert torch.equal(same, _call(a[:1].repeat(24, 1), b, None if sa is None else sa[:1].repeat(24, 1), sb, False))
        place = r.clone()
        assert _call(a, b, sa, sb, False, residual=place, out=place, **k) is place and torch.equal(place, want)
        with monkeypatch.context() as m:
            m.setattr(_lib, "_host", _lib._NoHost())
            assert torch.equal(_call(a, b, sa, sb, False, residual=r, **k), want)


def test_far_rows():
    """Rows further apart than the kernels take are laid out first."""
    store = torch.zeros(3, 3 << 20, dtype=torch.bfloat16, device="cuda")
    g, (a, b, _, _) = _case(torch.bfloat16, 3, 64, 128)
    store[:, :128] = a
    assert torch.equal(_call(store[:, :128], b, None, None, False), _call(a, b, None, None, False))


@pytest.mark.parametrize("M", [24, 200])
def test_in_place_and_overlaps(M):
    g, (a, b, _, _) = _case(torch.bfloat16, M, 256, 256)
    r = _normal(g, M, 256).to(torch.bfloat16)
    want = _call(a, b, None, None, False, residual=r)
    room = torch.zeros(M + 1, 256, dtype=torch.bfloat16, device="cuda")
    room[:M] = r
    with pytest.raises(RuntimeError, match="overlaps"):
        _call(a, b, None, None, False, residual=room[:M], out=room[1:])
    assert torch.equal(_call(a, b, None, None, False, residual=room[:M], out=room[:M]), want)
    for bad in (dict(out=a[:, :256]), dict(residual=r, out=b[:M]) if M <= 256 else dict(out=a)):
        with pytest.raises(RuntimeError, match="overlaps"):
            _call(a, b, None, None, False, **bad)


def test_refusals():
    from lightop_amd import gemmopt

    g, (a, b, _, _) = _case(torch.bfloat16, 8, 64, 128)
    _, (i, j, si, sj) = _case(torch.int8, 8, 64, 128)
    f = torch.zeros(64, device="cuda")
    bad = [lambda: gemmopt.gemm_bias_act(a.float(), b.float()), lambda: gemmopt.gemm_bias_act(a, b.half()), lambda: gemmopt.gemm_bias_act(a, b[:, :64]),
           lambda: gemmopt.gemm_bias_act(a[:, :4], b[:, :4]), lambda: gemmopt.gemm_bias_act(a, b, bias=f[:63]), lambda: gemmopt.gemm_bias_act(a, b, bias=f.half()),
           lambda: gemmopt.gemm_bias_act(a, b, bias=f.double()), lambda: gemmopt.gemm_bias_act(a, b, residual=f.bfloat16()),
           lambda: gemmopt.gemm_bias_act(a, b, residual=f.expand(8, 64)), lambda: gemmopt.gemm_bias_act(a, b, out_dtype=torch.float64),
           lambda: gemmopt.gemm_bias_act(a, b, out=torch.empty(8, 64, device="cuda")), lambda: gemmopt.gemm_bias_act(a, b.cpu()),
           lambda: gemmopt.gemm_bias_act(a, b, out=torch.empty(64, 8, dtype=a.dtype, device="cuda").t()), lambda: gemmopt.gemm_bias_act(a[:, :0], b[:, :0]),
           lambda: gemmopt.gemm_act_and_mul(a, b[:63]), lambda: gemmopt.gemm_w8a8_bias_act(a, b, si, sj), lambda: gemmopt.gemm_w8a8_bias_act(i, j, si[:7], sj),
           lambda: gemmopt.gemm_w8a8_bias_act(i, j, si, sj[:63]), lambda: gemmopt.gemm_w8a8_bias_act(i, j, si.half(), sj),
           lambda: gemmopt.gemm_w8a8_bias_act(i, j, None, None), lambda: gemmopt.gemm_w8a8_act_and_mul(i, j, si, None),
           lambda: gemmopt.gemm_w8a8_bias_act(i[:, :120], j[:, :120], si, sj), lambda: gemmopt.gemm_bias_act(i, j),
           lambda: gemmopt.gemm_w8a8_bias_act(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), torch.zeros(1, 131072, dtype=torch.int8, device="cuda"),
                                              si[:1], sj[:1])]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: gemmopt.gemm_bias_act(a, b, activation="relu"), lambda: gemmopt.gemm_act_and_mul(a, b, activation=None),
                 lambda: gemmopt.gemm_w8a8_act_and_mul(i, j, si, sj, activation="tanh")):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("M", [1, 4, 60, 300])
def test_streams_and_graphs(kind, M):
    g, (a, b, sa, sb) = _case(kind, M, 640, 1024)
    r = _normal(g, M, 640).to(_out(kind, None))
    want = _call(a, b, sa, sb, False, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _call(a, b, sa, sb, False, residual=r)
    side.synchronize()
    assert torch.equal(got, want)
    x, total = a.clone(), r.clone()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append((_call(x, b, sa, sb, False, residual=total), _call(x, b, sa, sb, True, out_dtype=torch.float32)))
    for k in range(4):
        x.copy_(a.roll(k + 1, 0 if M > 1 else 1))
        total.copy_(r * k)
        graphs[k & 1].replay()
        graphs[1 - (k & 1)].replay()
        eager = _call(x, b, sa, sb, False, residual=total), _call(x, b, sa, sb, True, out_dtype=torch.float32)
        torch.cuda.synchronize()
        for pair in outs:
            assert torch.equal(pair[0], eager[0]) and torch.equal(pair[1], eager[1])


def test_threads():
    """Sizes whose parts go through scratch, from two threads on one stream and one on another."""
    import threading

    sets = [_case(torch.bfloat16, 60, 576, 7168)[1], _case(torch.int8, 333, 576, 7168)[1]]
    want = [_call(*s, False) for s in sets]
    torch.cuda.synchronize()
    made = {}

    def work(name, stream):
        with torch.cuda.stream(stream):
            made[name] = [_call(*sets[i % 2], False) for i in range(40)]
            stream.synchronize()

    main = torch.cuda.current_stream()
    threads = [threading.Thread(target=work, args=(n, s)) for n, s in (("own", torch.cuda.Stream()), ("same", main), ("too", main))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 3
    for outs in made.values():
        assert len(outs) == 40 and all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs))


@pytest.mark.parametrize("kind,M,N,K,gated", [(torch.bfloat16, 20, 576, 7168, False), (torch.float16, 333, 577, 7168, False),
                                              (torch.int8, 20, 288, 7168, True), (torch.int8, 130, 300, 16384, False), (torch.bfloat16, 333, 289, 4096, True)])
def test_without_room_for_parts(kind, M, N, K, gated):
    """The C entry point with no workspace, and with one that is too small by a byte: K in one piece."""
    from lightop_amd import _lib

    g, (a, b, sa, sb) = _case(kind, M, 2 * N if gated else N, K)
    lib, code = _lib.lib(), {torch.bfloat16: 0, torch.float16: 1, torch.int8: 3}[kind]
    need = lib.lo_gemm_bias_act_workspace_bytes(code, int(gated), M, N, K)
    assert need >= 0
    room = torch.full((need + 256,), 0xff, dtype=torch.uint8, device="cuda")
    want = ref.dense(a, b, sa, sb, activation="silu" if gated else None, gated=gated)
    for n in sorted({0, max(need - 1, 0), need}):
        out = torch.empty(M, N, dtype=torch.float32, device="cuda")
        _lib.check(lib.lo_gemm_bias_act(_lib.ptr(a), K, _lib.ptr(b), K, code, _lib.ptr(sa), _lib.ptr(sb), None, 0, 0 if gated else -1, int(gated), 1.0,
                                        None, 0, _lib.ptr(out), 2, M, N, K, _lib.ptr(room if n else None), n, _lib.stream_of(a)))
        ref.check(out, want)
    assert (room[need:] == 0xff).all()
