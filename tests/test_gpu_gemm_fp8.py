"""Dense e4m3 product with block scales against float64."""
import ctypes

import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu


def _make(M, N, K, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + M * 7 + N * 3 + K)
    quotient, s = ref.groups_fp8(ref.rows(M, K, g, "cuda").double())
    b, bs = ref.weights((N, K), g, "cuda")
    return quotient.float().to(ref.FP8), b, s.float(), bs


def _bound(a, b, sa, sb, dtype, exact):
    """An e4m3 instruction is off by at most 2^-11 of the block's largest product (the bits of the others that it keeps), the exact one by
    fp32 roundings of 128 products; K / 128 fp32 steps on top, and half a step of the output."""
    KB = a.shape[1] // 128
    tops = lambda t: t.double().abs().unflatten(-1, (-1, 128)).amax(-1)
    rows = sb.double().repeat_interleave(128, 0)[:b.shape[0]]
    spread = (a.double().abs().unflatten(-1, (-1, 128)) * sa.double().unsqueeze(-1)).flatten(-2) @ ref.dequant(b.float().abs(), rows).T
    off = spread * (KB + 132 + 4) * ref.ULP32
    if dtype != torch.float32:
        off = off + 2.0 ** -11 * ((tops(a) * sa.double()) @ (tops(b) * rows).T)
    return off + 1.01 * ref.half_step(dtype, exact)


def _check(out, a, b, sa, sb):
    exact = ref.dequant(a, sa) @ ref.dequant_weight(b, sb).T
    assert out.shape == exact.shape
    assert ((out.double() - exact).abs() <= _bound(a, b, sa, sb, out.dtype, exact)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 48, 64, 65, 100, 128, 129, 200, 257, 400, 777])
@pytest.mark.parametrize("N,K", [(1, 128), (17, 384), (128, 1024), (576, 2048), (1001, 640), (2048, 768)])
def test_sizes(dtype, M, N, K):
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    print("[case] gemm", dtype, M, N, K, flush=True)
    a, b, sa, sb = _make(M, N, K)
    _check(gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=dtype), a, b, sa, sb)


@pytest.mark.parametrize("M,N,K", [(1, 4096, 7168), (48, 7168, 2048), (333, 576, 7168), (1531, 7168, 2048), (4099, 4096, 1152), (300, 264, 16384),
                                   (2048, 2048, 2048)])
def test_full_sizes(M, N, K):
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    print("[case] gemm", M, N, K, flush=True)
    a, b, sa, sb = _make(M, N, K)
    out = gemm_w8a8_fp8_block(a, b, sa, sb)
    _check(out, a, b, sa, sb)
    assert torch.equal(out, gemm_w8a8_fp8_block(a, b, sa, sb))  # one order of the sum


@pytest.mark.parametrize("M", [3, 40, 70, 300, 600])
@pytest.mark.parametrize("N", [40, 250, 520])
def test_nothing_else_is_written_and_nans_stay_in_their_row(M, N):
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    a, b, sa, sb = _make(M, N, 512)
    room = torch.full((M * N + 4096,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = room[2048:2048 + M * N].view(M, N)
    want = gemm_w8a8_fp8_block(a, b, sa, sb)
    got = gemm_w8a8_fp8_block(a, b, sa, sb, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
    assert (room[:2048] == 7).all() and (room[2048 + M * N:] == 7).all()
    nan = torch.tensor(float("nan"), device="cuda").to(ref.FP8)
    a, b = a.clone(), b.clone()
    a.view(torch.uint8)[M - 1, 5] = nan.view(torch.uint8)
    b.view(torch.uint8)[N - 1, 200] = nan.view(torch.uint8)
    got = gemm_w8a8_fp8_block(a, b, sa, sb)
    assert got[M - 1].isnan().all() and got[:, N - 1].isnan().all() and torch.equal(got[:-1, :-1], want[:-1, :-1])
    sa = sa.clone()
    sa[0, 1] = float("inf")
    assert (~got[1:-1, :-1].isnan()).all() and (~gemm_w8a8_fp8_block(a, b, sa, sb)[0].isfinite()).all()


def test_zero_rows_and_columns():
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    a, b, sa, sb = _make(70, 130, 256)
    assert gemm_w8a8_fp8_block(a[:0], b, sa[:0], sb).shape == (0, 130)
    assert gemm_w8a8_fp8_block(a, b[:0], sa, sb[:0]).shape == (70, 0)
    zero = torch.zeros_like(a.float()).to(ref.FP8)
    assert (gemm_w8a8_fp8_block(zero, b, torch.zeros_like(sa), sb) == 0).all()


@pytest.mark.parametrize("M,N,K", [(310000, 24, 7168), (40, 310000, 7168), (70000, 16384, 128)])
def test_offsets_past_32_bits(M, N, K):
    """Operands and results of more than 2 GiB: the last rows and columns."""
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    print("[case] gemm", M, N, K, flush=True)
    g = torch.Generator(device="cuda").manual_seed(5)

    def codes(n):
        return torch.randint(0, 0x7f, (n, K), generator=g, dtype=torch.uint8, device="cuda").view(ref.FP8)

    a, b = codes(M), codes(N)
    sa = torch.rand(M, K // 128, generator=g, device="cuda") * 1e-3
    sb = torch.rand(-(-N // 128), K // 128, generator=g, device="cuda") * 1e-3
    out = gemm_w8a8_fp8_block(a, b, sa, sb)
    m, n = min(M, 200), min(N, 128 + N % 128)
    m0, n0 = M - m, (N - n) // 128 * 128
    _check(out[m0:, n0:], a[m0:], b[n0:], sa[m0:], sb[n0 // 128:])
    _check(out[:m, :n], a[:m], b[:n], sa[:m], sb[:-(-n // 128)])


def test_strides_batches_and_marshalling(monkeypatch):
    from lightop_amd import _lib
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    a, b, sa, sb = _make(24, 96, 256)
    want = gemm_w8a8_fp8_block(a, b, sa, sb)
    got = gemm_w8a8_fp8_block(a.view(2, 12, 256), b, sa.view(2, 12, 2), sb)
    assert got.shape == (2, 12, 96) and torch.equal(got.view(24, 96), want)
    off = torch.zeros(24 * 256 + 1, dtype=torch.uint8, device="cuda")[1:].view(24, 256).copy_(a.view(torch.uint8)).view(ref.FP8)
    turned = sa.t().contiguous().t()
    assert torch.equal(gemm_w8a8_fp8_block(off, b, turned, sb), want)
    wide = torch.zeros(96, 512, dtype=torch.uint8, device="cuda").view(ref.FP8)
    wide.view(torch.uint8)[:, 256:] = b.view(torch.uint8)
    assert torch.equal(gemm_w8a8_fp8_block(a, wide[:, 256:], sa, sb), want)
    monkeypatch.setattr(_lib, "_host", _lib._NoHost())
    assert torch.equal(gemm_w8a8_fp8_block(a, b, sa, sb), want)
    for bad in (lambda: gemm_w8a8_fp8_block(a.float(), b, sa, sb), lambda: gemm_w8a8_fp8_block(a, b[:, :128], sa, sb),
                lambda: gemm_w8a8_fp8_block(a, b, sa[:, :1], sb), lambda: gemm_w8a8_fp8_block(a, b, sa, sb.double()),
                lambda: gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=torch.float64), lambda: gemm_w8a8_fp8_block(a, b, sa, sb.cpu()),
                lambda: gemm_w8a8_fp8_block(a, b, sa, sb, out=want[:, :90]), lambda: gemm_w8a8_fp8_block(a[:, :64], b[:, :64], sa, sb)):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("M", [4, 60, 300])
def test_streams_and_graphs(M):
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    a, b, sa, sb = _make(M, 640, 1024)
    want = gemm_w8a8_fp8_block(a, b, sa, sb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gemm_w8a8_fp8_block(a, b, sa, sb)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    sx = sa.clone()
    with torch.cuda.graph(graph):
        one = gemm_w8a8_fp8_block(a, b, sx, sb)
        two = gemm_w8a8_fp8_block(a, b, sx, sb, out_dtype=torch.float32)
    for k in range(3):
        sx.copy_(sa * (k + 1))
        graph.replay()
        eager = gemm_w8a8_fp8_block(a, b, sa * (k + 1), sb), gemm_w8a8_fp8_block(a, b, sa * (k + 1), sb, out_dtype=torch.float32)
        torch.cuda.synchronize()
        assert torch.equal(one, eager[0]) and torch.equal(two, eager[1])


@pytest.mark.parametrize("M,N,K", [(20, 576, 7168), (333, 576, 7168), (333, 577, 4096), (333, 577, 7168), (600, 4096, 7168), (130, 300, 16384)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_without_room_for_parts(M, N, K, dtype):
    """The C entry point with no workspace, and with one that is too small by a byte: K in one piece.  (Which sizes are split
    differs by the output's type; the smallest and narrowest are.)"""
    from lightop_amd import _lib

    a, b, sa, sb = _make(M, N, K)
    lib, code = _lib.lib(), {torch.bfloat16: 0, torch.float32: 2}[dtype]
    need = lib.lo_gemm_w8a8_fp8_block_workspace_bytes(M, N, K, code)
    assert need > 0 or M * N > 150000
    room = torch.full((need + 256,), 0xff, dtype=torch.uint8, device="cuda")
    outs = []
    for n in sorted({0, max(need - 1, 0), need}):
        out = torch.empty(M, N, dtype=dtype, device="cuda")
        _lib.check(lib.lo_gemm_w8a8_fp8_block(_lib.ptr(a), _lib.ptr(sa), _lib.ptr(b), _lib.ptr(sb), _lib.ptr(out), code, M, N, K,
                                              _lib.ptr(room if n else None), n, _lib.stream_of(a)))
        _check(out, a, b, sa, sb)
        outs.append(out)
    assert (room[need:] == 0xff).all()


def test_threads():
    """Sizes whose parts go through scratch, from two threads on one stream and one on another."""
    import threading

    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    sets = [_make(n, 576, 7168) for n in (60, 333)]
    want = [gemm_w8a8_fp8_block(a, b, sa, sb) for a, b, sa, sb in sets]
    torch.cuda.synchronize()
    made = {}

    def work(name, stream):
        with torch.cuda.stream(stream):
            made[name] = []
            for i in range(40):
                a, b, sa, sb = sets[i % 2]
                made[name].append(gemm_w8a8_fp8_block(a, b, sa, sb))
            stream.synchronize()

    main = torch.cuda.current_stream()
    threads = [threading.Thread(target=work, args=(n, s)) for n, s in (("own", torch.cuda.Stream()), ("same", main), ("too", main))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs in made.values():
        assert len(outs) == 40 and all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs))


@pytest.mark.parametrize("M,N,K", [(3990, 4001, 8448), (3990, 4002, 1152), (2001, 5003, 1152), (1337, 7003, 2048), (1337, 7004, 8576),
                                   (1300, 3333, 2048), (557, 3999, 7168), (563, 4001, 9216), (479, 7001, 8320), (82, 4097, 7168), (90, 4003, 9088),
                                   (150, 3001, 8320), (110, 2051, 8320), (3310, 577, 7168)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_ragged_products_of_every_tile(dtype, M, N, K):
    """Each tile, whole and in parts, with rows and columns that end inside it, rows of the result that begin off 16 bytes, more than 64 K
    blocks (the weights' scales come 64 at a time) and numbers of them that are no multiple of four."""
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    print("[case] gemm", dtype, M, N, K, flush=True)
    a, b, sa, sb = _make(M, N, K)
    out = gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=dtype)
    _check(out, a, b, sa, sb)
    assert torch.equal(out, gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=dtype))


@pytest.mark.parametrize("M,N,K", [(7, 64, 256), (333, 576, 7168), (20, 576, 7168), (300, 264, 384), (300, 2048, 2048)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_an_output_that_begins_on_any_value(dtype, M, N, K, shift):
    """Columns in fours, and an `out` that begins off 8 and 16 bytes: up to 16 rows, in parts of K and whole."""
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    print("[case] gemm", dtype, M, N, K, shift, flush=True)
    a, b, sa, sb = _make(M, N, K)
    room = torch.full((M * N + 64,), 7.0, dtype=dtype, device="cuda")
    out = room[32 + shift:32 + shift + M * N].view(M, N)
    assert out.data_ptr() % 8 or dtype == torch.float32
    gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=dtype, out=out)
    assert torch.equal(out, gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=dtype))
    _check(out, a, b, sa, sb)
    assert (room[:32 + shift] == 7).all() and (room[32 + shift + M * N:] == 7).all()


@pytest.mark.parametrize("M,N,K", [(20, 576, 7168), (130, 300, 16384), (333, 576, 7168), (333, 577, 7168)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_less_room_than_the_parts_take_is_no_room(dtype, M, N, K):
    """A workspace that is too small, by a byte or by half: the bits of a call without one, and nothing written to it."""
    from lightop_amd import _lib

    a, b, sa, sb = _make(M, N, K)
    lib, code = _lib.lib(), {torch.bfloat16: 0, torch.float32: 2}[dtype]
    need = lib.lo_gemm_w8a8_fp8_block_workspace_bytes(M, N, K, code)
    assert need > 0

    def run(n):
        out, room = torch.empty(M, N, dtype=dtype, device="cuda"), torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
        _lib.check(lib.lo_gemm_w8a8_fp8_block(_lib.ptr(a), _lib.ptr(sa), _lib.ptr(b), _lib.ptr(sb), _lib.ptr(out), code, M, N, K,
                                              _lib.ptr(room if n else None), n, _lib.stream_of(a)))
        return out, bool((room == 0xff).all())

    whole, untouched = run(0)
    assert untouched
    for n in (need - 1, need // 2, 16):
        out, untouched = run(n)
        assert untouched and torch.equal(out, whole), n
    out, untouched = run(need)
    assert not untouched
    _check(out, a, b, sa, sb)


@pytest.mark.parametrize("tile,size", ref.TILE_SIZES, ids=lambda v: "x".join(map(str, v)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_every_tile(dtype, tile, size):
    """Each tile, whole and in parts, with what ends inside it; without a workspace the tiles that K in one piece takes."""
    from lightop_amd import _lib
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    M, N, K = size
    lib, code = _lib.lib(), {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}[dtype]
    got = [ctypes.c_int32() for _ in range(3)]
    _lib.check(lib.lo_gemm_w8a8_fp8_block_tile_query(M, N, K, code, 1, *(ctypes.byref(v) for v in got)))
    m, n, parts = (v.value for v in got)
    assert dtype == torch.float32 or (m, n, parts > 1) == tile
    print("[case] gemm", dtype, M, N, K, "tile", m, n, parts, flush=True)
    a, b, sa, sb = _make(M, N, K)
    out = gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=dtype)
    _check(out, a, b, sa, sb)
    assert torch.equal(out, gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=dtype))
    if parts > 1:
        whole = torch.empty_like(out)
        _lib.check(lib.lo_gemm_w8a8_fp8_block(_lib.ptr(a), _lib.ptr(sa), _lib.ptr(b), _lib.ptr(sb), _lib.ptr(whole), code, M, N, K, None, 0,
                                              _lib.stream_of(a)))
        _check(whole, a, b, sa, sb)


@pytest.mark.parametrize("M,N,K", [(3, 250, 512), (70, 520, 512), (600, 250, 512), (20, 576, 7168), (333, 577, 7168)])
def test_infinite_scales_stay_in_their_rows_and_columns(M, N, K):
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    a, b, sa, sb = _make(M, N, K)
    want = gemm_w8a8_fp8_block(a, b, sa, sb)
    rows, cols = sa.clone(), sb.clone()
    rows[1, K // 128 - 1] = float("inf")
    cols[0, 2] = float("nan")
    got = gemm_w8a8_fp8_block(a, b, rows, sb)
    assert not got[1].isfinite().any() and torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:])
    got = gemm_w8a8_fp8_block(a, b, sa, cols)
    assert got[:, :128].isnan().all() and torch.equal(got[:, 128:], want[:, 128:])


def _eights(a, b, sa, rows):
    """Sum over K of the largest |product| of every eight that follow each other, with the scales."""
    pa = (a.double().abs().unflatten(-1, (-1, 128)) * sa.double().unsqueeze(-1)).flatten(-2).unflatten(-1, (-1, 8))
    pb = ref.dequant(b.double().abs(), rows).unflatten(-1, (-1, 8))
    return torch.stack([(pa[m].unsqueeze(0) * pb).amax(-1).sum(-1) for m in range(a.shape[0])])


def _hard(kind, M, N, K):
    """Operands whose eights hold products of very different sizes."""
    a, b, sa, sb = _make(M, N, K)
    x, y = a.float().clamp(-8, 8), b.float().clamp(-8, 8)
    if kind == "one sign":
        x, y = torch.full_like(x, 3.75), torch.full_like(y, 3.75)
        x[:, ::8], y[:, ::8] = 448.0, 448.0
    else:  # the largest products of each eight cancel
        x[:, ::8], y[:, ::8] = 448.0, 448.0
        x[:, 1::8], y[:, 1::8] = -448.0, 448.0
    return x.to(ref.FP8), y.to(ref.FP8), sa, sb


@pytest.mark.parametrize("kind", ["one sign", "cancelling"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("M,N,K", [(1, 300, 512), (16, 130, 2048), (17, 130, 2432), (40, 264, 512), (70, 300, 384)])
def test_products_of_very_different_sizes(kind, dtype, M, N, K):
    """fp32 roundings of the sum up to 16 tokens and in fp32.  Else the e4m3 instruction's: seven products of an eight lose less than 2^-13 of its
    largest each (the exponent of which is that of 2^(e_a + e_b) at least)."""
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    a, b, sa, sb = _hard(kind, M, N, K)
    rows = sb.double().repeat_interleave(128, 0)[:N]
    exact = ref.dequant(a, sa) @ ref.dequant_weight(b, sb).T
    spread = (a.double().abs().unflatten(-1, (-1, 128)) * sa.double().unsqueeze(-1)).flatten(-2) @ ref.dequant(b.double().abs(), rows).T
    off = spread * (K // 128 + 136) * ref.ULP32
    if M > 16 and dtype != torch.float32:
        off = off + 7 * 2.0 ** -13 * _eights(a, b, sa, rows)
    out = gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=dtype).double()
    assert ((out - exact).abs() <= off + 1.01 * ref.half_step(dtype, exact.abs() + off)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("M,N,K", [(8, 8200, 1024), (16, 4096, 7168), (48, 4096, 2048), (130, 1000, 7168), (700, 1000, 2048)])
def test_error_of_the_whole_result(dtype, M, N, K):
    """The norm of the error is that of rounding the exact result, with what the products lose: 1e-4 for the e4m3 instruction (some 2e-5 for rows
    like these), 1e-6 for the exact one (fp32 roundings, some of 150 of them, of 2^-24 each)."""
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    a, b, sa, sb = _make(M, N, K)
    exact = ref.dequant(a, sa) @ ref.dequant_weight(b, sb).T
    out = gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=dtype).double()
    rounding = (exact.to(dtype).double() - exact).norm()
    lost = 1e-6 if M <= 16 or dtype == torch.float32 else 1e-4
    assert (out - exact).norm() <= 1.01 * rounding + lost * exact.norm()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("M,N,K", [(1, 4096, 7168), (16, 2048, 2048), (7, 8200, 640)])
def test_up_to_16_tokens_only_fp32_roundings_are_in_front_of_the_output(dtype, M, N, K):
    """A result that is off by e in front of its rounding is another than the exact one's rounding in e / step of the cases: 1e-6, some 150 fp32
    roundings, against a step of eps times 0.7 of the value, and values below the mean; four times that allowed."""
    from lightop_amd.gemmopt import gemm_w8a8_fp8_block

    a, b, sa, sb = _make(M, N, K)
    exact = ref.dequant(a, sa) @ ref.dequant_weight(b, sb).T
    off = _bound(a, b, sa, sb, torch.float32, exact)
    out = gemm_w8a8_fp8_block(a, b, sa, sb, out_dtype=dtype)
    assert ((out.double() - exact).abs() <= off + ref.half_step(dtype, exact.abs() + off)).all()
    assert (out != exact.to(dtype)).double().mean() <= 4e-6 / torch.finfo(dtype).eps + 2 / out.numel()
