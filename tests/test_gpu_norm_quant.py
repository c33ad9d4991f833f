"""RMS norm with 8-bit output against its definition in float64, and against the package's quantisations of the fp32 normed rows."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu
FORMS = {"int8 rows": (torch.int8, None), "int8 groups": (torch.int8, 128), "fp8 groups": (torch.float8_e4m3fn, 128)}
# a row's sum of squares: up to 64 fused steps a thread and 10 across it, halved by the root; four more roundings; twice for value and maximum
REL = 2.0 ** -17


def _make(M, H, dtype, residual, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * M + H)
    x = ref.rows(M, H, g, "cuda", dtype)
    r = (4 * ref.rows(M, H, g, "cuda")).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(H, generator=g, device="cuda")).to(dtype)
    return x, r, w


def _check(out, x, r, w, form, eps, normed, rows=slice(None)):
    dtype = x.dtype
    z = x.double() if r is None else x.double() + r.double()
    y = z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps) * w.double()
    if r is None:
        assert out.residual is None
    else:
        assert out.residual.dtype == dtype and ((out.residual.double() - z).abs() <= 1.01 * ref.half_step(dtype, z)).all()
    if normed:
        assert ((out.normed.double() - y).abs() <= (1.01 + (REL * 2 / torch.finfo(dtype).eps)) * ref.half_step(dtype, y)).all()
    else:
        assert out.normed is None
    if form == "fp8 groups":
        quotient, scale = ref.groups_fp8(y)
        assert ((out.scale.double() - scale).abs() <= REL * scale).all()
        assert ref.codes_ok(out.q, quotient, REL)
        return
    v = y.unsqueeze(-2) if form == "int8 rows" else y.unflatten(-1, (-1, 128))
    scale = v.abs().amax(-1).clamp(min=1e-10) / 127
    assert out.scale.shape == scale.shape and ((out.scale.double() - scale).abs() <= REL * scale).all()
    t = (v / scale.unsqueeze(-1)).flatten(-2)
    off = out.q.double() - t
    if form == "int8 rows":  # nearest
        assert (off.abs() <= 0.5 + 127 * REL).all()
    else:                    # towards zero
        off = off * torch.where(t < 0, -1.0, 1.0)
        assert (off <= 127 * REL).all() and (off > -1 - 127 * REL).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("M,H", [(1, 128), (1, 2048), (3, 1024), (2, 640), (7, 7168), (5, 8192), (2, 8320), (3, 16384), (2, 16512), (2, 65536),
                                 (333, 896), (700, 4096)])
def test_values(form, dtype, M, H):
    from lightop_amd.norm import rms_norm_quant

    print("[case] norm", form, dtype, M, H, flush=True)
    for residual, normed in ((True, True), (False, False), (True, False)):
        x, r, w = _make(M, H, dtype, residual)
        if normed:
            w = w.float()  # the other weight type
        q, g = FORMS[form]
        out = rms_norm_quant(x, w, 1e-6, residual=r, quant_dtype=q, group_size=g, return_normed=normed)
        assert out.q.dtype == q and out.q.shape == x.shape
        _check(out, x, r, w, form, 1e-6, normed)


@pytest.mark.parametrize("H", [8, 72, 1000, 5000, 9000])
def test_rows_of_odd_widths(H):
    from lightop_amd.norm import rms_norm_quant

    x, r, w = _make(5, H, torch.bfloat16, True)
    _check(rms_norm_quant(x, w, 1e-5, residual=r), x, r, w, "int8 rows", 1e-5, False)


@pytest.mark.parametrize("form", FORMS)
def test_codes_are_those_of_the_fp32_rows(form):
    from lightop_amd.norm import rms_norm_quant
    from lightop_amd.quant import per_token_group_quant_fp8, per_token_group_quant_int8

    x, r, w = _make(37, 2048, torch.float32, True)
    q, g = FORMS[form]
    out = rms_norm_quant(x, w, residual=r, quant_dtype=q, group_size=g, return_normed=True)
    if form == "int8 rows":
        top = out.normed.abs().amax(-1, keepdim=True)
        # (tensors: torch divides by a host number through its reciprocal)
        n = torch.full_like(top, 127.0)
        assert torch.equal(out.scale, top / n)
        assert torch.equal(out.q, torch.round(out.normed * (n / top)).to(torch.int8))
        return
    want = (per_token_group_quant_int8 if form == "int8 groups" else per_token_group_quant_fp8)(out.normed, 128)
    assert torch.equal(out.q.view(torch.int8), want[0].view(torch.int8)) and torch.equal(out.scale, want[1])


def test_strides_shapes_and_in_place():
    from lightop_amd.norm import rms_norm_quant

    x, r, w = _make(6, 256, torch.bfloat16, True)
    want = rms_norm_quant(x, w, residual=r, return_normed=True)
    wide = torch.zeros(6, 384, dtype=x.dtype, device="cuda")
    wide[:, 128:] = x
    offs = torch.zeros(6 * 256 + 1, dtype=x.dtype, device="cuda")[1:].view(6, 256).copy_(r)  # not 16-byte aligned
    for a, b in ((wide[:, 128:], r), (x, offs), (x.t().contiguous().t(), r), (x.view(2, 3, 256), r.view(2, 3, 256)),
                 (wide.view(2, 3, 384)[..., 128:], r.view(2, 3, 256))):
        got = rms_norm_quant(a, w, residual=b, return_normed=True)
        for u, v in zip(got, want):
            assert u.shape[:-1] == a.shape[:-1] and torch.equal(u.reshape(v.shape), v)
    keep = r.clone()
    got = rms_norm_quant(x, w, residual=keep, residual_out=keep)
    assert got.residual.data_ptr() == keep.data_ptr() and torch.equal(keep, want.residual) and torch.equal(got.q, want.q)
    y = x.clone()
    got = rms_norm_quant(y, w, residual=r, residual_out=y)
    assert torch.equal(y, want.residual) and torch.equal(got.q, want.q) and torch.equal(got.scale, want.scale)
    empty = rms_norm_quant(x[:0], w, residual=r[:0], return_normed=True)
    assert empty.q.shape == (0, 256) and empty.scale.shape == (0, 1) and empty.residual.shape == empty.normed.shape == (0, 256)


@pytest.mark.parametrize("form", FORMS)
def test_special_rows(form):
    """A row of zeros, of the largest 16-bit values, of denormals; one with a NaN leaves its neighbours alone."""
    from lightop_amd.norm import rms_norm_quant

    q, g = FORMS[form]
    x, _, w = _make(5, 256, torch.float16, False)
    x[0] = 0
    x[1] = 65504
    x[2] = 6e-8
    x[3, 7] = float("nan")
    out = rms_norm_quant(x, w, 1e-6, quant_dtype=q, group_size=g)
    assert (out.q[0].float() == 0).all() and torch.equal(
        out.scale[0], torch.full_like(out.scale[0], 1e-10) / torch.full_like(out.scale[0], 448.0 if q != torch.int8 else 127.0))
    keep = [0, 1, 2, 4]
    part = type(out)(out.q[keep], out.scale[keep], None, None)
    _check(part, x[keep], None, w, form, 1e-6, False)


def test_python_marshalling_gives_the_same(monkeypatch):
    from lightop_amd import _lib
    from lightop_amd.norm import rms_norm_quant

    for form, (q, g) in FORMS.items():
        x, r, w = _make(9, 1024, torch.bfloat16, True)
        a = rms_norm_quant(x, w, residual=r, quant_dtype=q, group_size=g, return_normed=True)
        with monkeypatch.context() as m:
            m.setattr(_lib, "_host", _lib._NoHost())
            b = rms_norm_quant(x, w, residual=r, quant_dtype=q, group_size=g, return_normed=True)
        assert all(torch.equal(u.view(torch.int8), v.view(torch.int8)) for u, v in zip(a, b))


def test_refusals():
    from lightop_amd.norm import rms_norm_quant

    x, r, w = _make(4, 256, torch.bfloat16, True)
    for bad in (lambda: rms_norm_quant(x[:, :252], w[:252]), lambda: rms_norm_quant(x, w[:128]), lambda: rms_norm_quant(x, w.half()),
                lambda: rms_norm_quant(x, w, residual=r[:2]), lambda: rms_norm_quant(x, w, residual=r.half()),
                lambda: rms_norm_quant(x, w, residual_out=r), lambda: rms_norm_quant(x, w, residual=r, residual_out=r.t().contiguous().t()),
                lambda: rms_norm_quant(x.int(), w), lambda: rms_norm_quant(x, w.cpu()), lambda: rms_norm_quant(x, w, -1.0),
                lambda: rms_norm_quant(x[:, :0], w[:0]), lambda: rms_norm_quant(x, w, quant_dtype=torch.int8, group_size=64)):
        with pytest.raises(RuntimeError):
            bad()


def test_streams_and_graphs():
    from lightop_amd.norm import rms_norm_quant

    x, r, w = _make(65, 2048, torch.bfloat16, True)
    want = rms_norm_quant(x, w, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rms_norm_quant(x, w, residual=r)
    side.synchronize()
    assert torch.equal(got.q, want.q)
    graph = torch.cuda.CUDAGraph()
    sx = x.clone()
    with torch.cuda.graph(graph):
        out = rms_norm_quant(sx, w, residual=r)
    for seed in range(3):
        y = _make(65, 2048, torch.bfloat16, True, seed)[0]
        sx.copy_(y)
        graph.replay()
        eager = rms_norm_quant(y, w, residual=r)
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out[:3], eager[:3]))


def test_a_sum_over_other_rows_is_refused():
    from lightop_amd.norm import rms_norm_quant

    buf = torch.zeros(6, 256, dtype=torch.bfloat16, device="cuda")
    x, _, w = _make(5, 256, torch.bfloat16, False)
    for out in (buf[:5], buf[1:]):
        rms_norm_quant(x, w, residual=out, residual_out=out)
        with pytest.raises(RuntimeError, match="overlaps"):
            rms_norm_quant(x, w, residual=buf[1:] if out.data_ptr() == buf.data_ptr() else buf[:5], residual_out=out)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("M,H", [(769, 128), (1000, 1152), (769, 2048), (801, 4224), (1500, 7168), (769, 16512), (770, 65536)])
def test_values_of_many_rows(form, dtype, M, H):
    """More rows than take one piece a thread: two, four and eight of them, and 1024 threads for the longest rows."""
    from lightop_amd.norm import rms_norm_quant

    print("[case] norm", form, dtype, M, H, flush=True)
    q, g = FORMS[form]
    x, r, w = _make(M, H, dtype, True)
    _check(rms_norm_quant(x, w, 1e-5, residual=r, quant_dtype=q, group_size=g, return_normed=True), x, r, w, form, 1e-5, True)
    x, r, w = _make(M, H, dtype, False, 1)
    _check(rms_norm_quant(x, w, 1e-5, quant_dtype=q, group_size=g), x, r, w, form, 1e-5, False)


@pytest.mark.parametrize("form", FORMS)
def test_more_rows_than_a_launch_takes(form):
    """Offsets past 32 bits, in bytes and in values, and a second launch: the rows around its first and the last ones."""
    from lightop_amd.norm import RmsNormQuant, rms_norm_quant

    M, H = 2 ** 21 + 700, 1032 if form == "int8 rows" else 1152
    q, g = FORMS[form]
    tile = torch.randn(4096, H, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(torch.bfloat16)
    x = tile.repeat(-(-M // 4096), 1)[:M]
    x[-5:] *= 3
    w = torch.ones(H, dtype=torch.bfloat16, device="cuda")
    out = rms_norm_quant(x, w, 1e-6, residual=x, quant_dtype=q, group_size=g)
    for part in (slice(0, 300), slice(2 ** 21 - 300, 2 ** 21 + 300), slice(M - 300, M)):
        _check(RmsNormQuant(out.q[part], out.scale[part], out.residual[part], None), x[part], x[part], w, form, 1e-6, False)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_a_sum_that_begins_on_any_value(form, dtype):
    """`residual_out` off 16 bytes: the residual itself, updated in place, and memory of its own, with nothing else written."""
    from lightop_amd.norm import rms_norm_quant

    q, g = FORMS[form]
    x, r, w = _make(7, 384, dtype, True)
    want = rms_norm_quant(x, w, residual=r, quant_dtype=q, group_size=g)
    for own in (True, False):
        room = torch.full((7 * 384 + 16,), 7.0, dtype=dtype, device="cuda")
        out = room[1:1 + 7 * 384].view(7, 384)
        assert out.data_ptr() % 16
        if own:
            out.copy_(r)
        got = rms_norm_quant(x, w, residual=out if own else r, residual_out=out, quant_dtype=q, group_size=g)
        assert got.residual is out and torch.equal(out, want.residual)
        assert torch.equal(got.q.view(torch.int8), want.q.view(torch.int8)) and torch.equal(got.scale, want.scale)
        assert room[0] == 7 and (room[1 + 7 * 384:] == 7).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("M", [4, 800])
def test_a_row_with_a_nan_or_an_infinity(form, M):
    """What becomes of the row itself: the codes and scales that the package's own quantisation gives its normed rows."""
    from lightop_amd.norm import rms_norm_quant
    from lightop_amd.quant import per_token_group_quant_fp8, per_token_group_quant_int8, per_token_quant_int8

    q, g = FORMS[form]
    x, _, w = _make(M, 256, torch.bfloat16, False)
    x[1, 7], x[2, 9] = float("nan"), float("-inf")
    out = rms_norm_quant(x, w, quant_dtype=q, group_size=g, return_normed=True)
    assert out.normed[1].isnan().all() and out.normed[2].isnan().sum() == 1 and (out.normed[2, 10:] == 0).all()
    rows = out.normed[1:3].contiguous()
    want = (per_token_quant_int8(rows) if form == "int8 rows" else
            (per_token_group_quant_int8 if form == "int8 groups" else per_token_group_quant_fp8)(rows, 128))
    assert torch.equal(out.q[1:3].view(torch.int8), want[0].view(torch.int8)) and torch.equal(out.scale[1:3], want[1])
    assert (out.scale[1:3] < 1e-12).all()
    if q == torch.int8:
        assert (out.q[1] == -128).all() and out.q[2, 9] == -128 and (out.q[2] == 0).sum() == 255
    else:
        assert out.q[1].float().isnan().all() and out.q[2].float().isnan().sum() == 1
    clean = x.clone()
    clean[1:3] = 1
    rest = rms_norm_quant(clean, w, quant_dtype=q, group_size=g)
    keep = [0, *range(3, M)]
    assert torch.equal(out.q[keep].view(torch.int8), rest.q[keep].view(torch.int8)) and torch.equal(out.scale[keep], rest.scale[keep])
