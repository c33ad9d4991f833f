"""Dense products in parts of K: their workspace on streams, in graphs and between threads, and the joining launch's ways out."""
import threading

import pytest
import torch

import dense_parts as parts
import dense_ref as ref

pytestmark = pytest.mark.gpu


def _call(a, b, sa, sb, gated, **k):
    from lightop_amd import gemmopt

    if sa is None:
        return (gemmopt.gemm_act_and_mul if gated else gemmopt.gemm_bias_act)(a, b, **k)
    return (gemmopt.gemm_w8a8_act_and_mul if gated else gemmopt.gemm_w8a8_bias_act)(a, b, sa, sb, **k)


def _case(size, seed=0):
    kind, M, N, K, gated = size
    parts.needs(*size)
    print("[case] parts", kind, M, N, K, gated, flush=True)
    g = torch.Generator(device="cuda").manual_seed(seed + M * 7 + N * 3 + K)
    return g, ref.operands(kind, M, 2 * N if gated else N, K, g)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _out(kind):
    return torch.bfloat16 if kind == torch.int8 else kind


@pytest.mark.parametrize("size", parts.PARTS, ids=str)
def test_every_way_out_of_the_joining_launch(size):
    """Biases, activations, residuals contiguous, strided and in place, every result's type; the same bits each time."""
    kind, M, N, K, gated = size
    g, ops = _case(size)
    rows = 2 * N if gated else N
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        if gated:
            for bias, name in ((None, "gelu"), (_normal(g, rows).to(dtype), "silu")):
                out = _call(*ops, True, bias=bias, activation=name, out_dtype=dtype)
                ref.check(out, ref.dense(*ops, bias, name, True))
                assert torch.equal(out, _call(*ops, True, bias=bias, activation=name, out_dtype=dtype))
            continue
        wide = _normal(g, M, N + 24).to(dtype)
        for bias, name, r, scale in ((_normal(g, rows), "silu", wide[:, :N].contiguous(), 0.75), (None, None, wide[:, 8:N + 8], -1.0),
                                     (_normal(g, rows).to(dtype), "gelu", wide[:, 3:N + 3], 1.0)):
            out = _call(*ops, False, bias=bias, activation=name, residual=r, scale=scale, out_dtype=dtype)
            ref.check(out, ref.dense(*ops, bias, name, False, r, scale))
            place = r.clone(memory_format=torch.contiguous_format)
            assert _call(*ops, False, bias=bias, activation=name, residual=place, scale=scale, out_dtype=dtype, out=place) is place
            assert torch.equal(place, out)


@pytest.mark.parametrize("size", parts.PARTS, ids=str)
def test_nothing_else_is_written_or_read(size):
    """Operands within wider tensors of NaNs (int8: of 127), values around the result, NaNs of a row and of a column."""
    kind, M, N, K, gated = size
    g, (a, b, sa, sb) = _case(size, 1)
    want = _call(a, b, sa, sb, gated)
    wide = [torch.full((t.shape[0] + 2, K + 80), 127 if kind == torch.int8 else float("nan"), dtype=kind, device="cuda") for t in (a, b)]
    for w, t in zip(wide, (a, b)):
        w[1:-1, 32:32 + K] = t
    room = torch.full((M * N + 4096,), 7.0, dtype=want.dtype, device="cuda")
    out = room[2048:2048 + M * N].view(M, N)
    _call(wide[0][1:-1, 32:32 + K], wide[1][1:-1, 32:32 + K], sa, sb, gated, out=out)
    assert torch.equal(out, want) and (room[:2048] == 7).all() and (room[2048 + M * N:] == 7).all()
    if kind == torch.int8:
        sa, sb = sa.clone(), sb.clone()
        sa[M - 1], sb[N - 1] = float("nan"), float("nan")
    else:
        a, b = a.clone(), b.clone()
        a[M - 1, 5], b[N - 1, K - 3] = float("nan"), float("nan")
    got = _call(a, b, sa, sb, gated)
    assert got[M - 1].isnan().all() and got[:, N - 1].isnan().all() and torch.equal(got[:-1, :-1], want[:-1, :-1])


@pytest.mark.parametrize("size", parts.PARTS, ids=str)
def test_without_room_for_parts(size):
    """The C entry point without a workspace, with one that is too small by a byte (both: K in one piece, the same bits) and with one that is just
    large enough, which is all that it writes to."""
    from lightop_amd import _lib

    kind, M, N, K, gated = size
    g, (a, b, sa, sb) = _case(size, 2)
    lib, need = _lib.lib(), parts.needs(*size)
    room = torch.full((need + 4096,), 0xa5, dtype=torch.uint8, device="cuda")
    want, made = ref.dense(a, b, sa, sb, activation="silu" if gated else None, gated=gated), {}
    for n in (0, need - 1, need):
        made[n] = torch.empty(M, N, dtype=torch.float32, device="cuda")
        _lib.check(lib.lo_gemm_bias_act(_lib.ptr(a), K, _lib.ptr(b), K, parts.CODES[kind], _lib.ptr(sa), _lib.ptr(sb), None, 0, 0 if gated else -1,
                                        int(gated), 1.0, None, 0, _lib.ptr(made[n]), 2, M, N, K, _lib.ptr(room[1024:] if n else None), n, _lib.stream_of(a)))
        ref.check(made[n], want)
        whole = (room == 0xa5).all()
        assert whole if n < need else not whole
    assert torch.equal(made[0], made[need - 1]) and torch.equal(made[need], _call(a, b, sa, sb, gated, out_dtype=torch.float32))
    assert (room[:1024] == 0xa5).all() and (room[1024 + need:] == 0xa5).all()


def test_side_streams():
    """Several calls of other sizes queued on two streams at a time, each with a workspace of its own that grows on the way."""
    sizes = sorted(parts.PARTS, key=lambda s: parts.needs(*s))
    sets = [(_case(s, 3)[1], s[4]) for s in sizes]
    want = [_call(*ops, gated) for ops, gated in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    made = {}
    for turn in range(6):
        for i, (ops, gated) in enumerate(sets):
            for j, s in enumerate(streams):
                with torch.cuda.stream(s):
                    made[turn, i, j] = _call(*ops, gated)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i]) for (_, i, _), out in made.items())


@pytest.mark.parametrize("shared", [False, True], ids=["own pools", "one pool"])
def test_graphs(shared):
    """Two graphs of several sizes each, replayed in turn over changing inputs with the program's own calls between, and residuals in place."""
    sets = []
    for i, s in enumerate(parts.PARTS):
        g, ops = _case(s, 4)
        sets.append((s, [None if t is None else t.clone() for t in ops], None if s[4] else _normal(g, s[1], s[2]).to(_out(s[0]))))
    totals = [None if r is None else torch.empty_like(r) for _, _, r in sets]

    def run(which, totals):
        outs = []
        for i in which:
            (kind, M, N, K, gated), ops, r = sets[i]
            if gated:
                outs.append(_call(*ops, True, activation="gelu"))
            else:
                totals[i].copy_(r)
                _call(*ops, False, residual=totals[i], out=totals[i])
                outs.append(_call(*ops, False, residual=totals[i], scale=0.5))
        return outs

    halves = [(0, 2, 4, 6), (1, 3, 5, 7)]
    run(halves[0] + halves[1], totals)
    torch.cuda.synchronize()
    graphs, made = [], []
    for which in halves:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if shared and len(graphs) > 1 else None):
            made.append(run(which, totals))
    for turn in range(4):
        for _, ops, _ in sets:
            ops[0].copy_(ops[0].roll(1, 0))
        for h in ((0, 1) if turn % 2 else (1, 0)):
            graphs[h].replay()
            got = [t.clone() for t in made[h]]
            want = run(halves[h], [None if t is None else torch.empty_like(t) for t in totals])
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want)), (turn, h)


def test_threads():
    """Workspaces of several sizes wanted on one stream by two threads at a time, and on another stream by a third one."""
    order = [0, 1, 3, 4]
    sets = [(_case(parts.PARTS[i], 5)[1], parts.PARTS[i][4]) for i in order]
    assert len({parts.needs(*parts.PARTS[i]) for i in order}) == len(order)
    want = [_call(*ops, gated) for ops, gated in sets]
    torch.cuda.synchronize()
    made, same = {}, torch.cuda.Stream()

    def work(name, stream, turned):
        with torch.cuda.stream(stream):
            made[name] = [(i, _call(*sets[i][0], sets[i][1])) for i in ((k * turned) % len(sets) for k in range(60))]
            stream.synchronize()

    threads = [threading.Thread(target=work, args=a) for a in (("own", torch.cuda.Stream(), 1), ("same", same, 1), ("too", same, 3))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 3
    for outs in made.values():
        assert len(outs) == 60 and all(torch.equal(o, want[i]) for i, o in outs)


@pytest.mark.parametrize("M,N,K", parts.WIDE)
def test_wide_tiles_in_parts(M, N, K):
    """Tiles of 128 x 256, plain, in parts: ragged tokens, columns and K."""
    for kind, out, k in ((torch.bfloat16, torch.bfloat16, K), (torch.float16, torch.float32, K), (torch.int8, torch.float16, 2 * K), (torch.int8, torch.float32, 2 * K)):
        g, ops = _case((kind, M, N, k, False), 6)
        more = dict(bias=_normal(g, N).to(out), activation="silu", residual=_normal(g, M, N).to(out), scale=0.75)
        got = _call(*ops, False, out_dtype=out, **more)
        ref.check(got, ref.dense(*ops, gated=False, **more))
        assert torch.equal(got, _call(*ops, False, out_dtype=out, **more))


PLAIN_TILES = [(tile, size) for tile, sizes in ref.TILES.items() if not tile[3] for size in sizes[:1]] + [((128, 256, True, False), parts.WIDE[0])]


@pytest.mark.parametrize("tile,size", PLAIN_TILES, ids=str)
def test_strided_residuals_of_every_tile(tile, size):
    """Residual rows further apart than the result's: on 16 bytes, where they are added in whole pieces, and off them, beside a result whose rows are on
    them; with values around the residual that would show."""
    M, N, K = size
    assert N % 8 == 0
    for kind, out, k in ((torch.bfloat16, torch.bfloat16, K), (torch.float16, torch.float32, K), (torch.int8, torch.float16, 2 * K)):
        print("[case] strided residual", tile, kind, M, N, k, flush=True)
        assert parts.plan(kind, M, N, k, False)[:2] == tile[:2]
        g = torch.Generator(device="cuda").manual_seed(M + N + k)
        ops = ref.operands(kind, M, N, k, g)
        r = _normal(g, M, N).to(out)
        want = _call(*ops, False, residual=r, scale=-0.5, out_dtype=out)
        ref.check(want, ref.dense(*ops, residual=r, scale=-0.5))
        for left, more in ((8, 24), (16, 16), (5, 24), (8, 27)):
            wide = torch.full((M, N + more), float("nan"), dtype=out, device="cuda")
            view = wide[:, left:left + N].copy_(r)
            assert torch.equal(_call(*ops, False, residual=view, scale=-0.5, out_dtype=out), want)
