"""The norms on both sides of a block, with gate and residual scale, against float64."""
import pytest
import torch

import fp8_ref
from fp8_ref import ULP32, half_step

pytestmark = pytest.mark.gpu

FORMS = [None, (torch.int8, None), (torch.int8, 128), (torch.float8_e4m3fn, 128)]


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _make(M, H, dtype, gate, post, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * M + H)
    x, r = _normal(g, M, H).to(dtype), (4 * _normal(g, M, H)).to(dtype)
    w = (1 + 0.2 * _normal(g, H)).to(dtype)
    p = (1 + 0.2 * _normal(g, H)) if post else None  # fp32 beside rows of any type
    shape = {None: None, "token": (M, 1), "channel": (H,), "full": (M, H)}[gate]
    return x, r, w, p, None if shape is None else _normal(g, *shape).to(dtype)


def _exact(x, r, w, p, gate, sigmoid, scale, residual_scale, eps):
    """z, y and their distance from an fp32 evaluation.  Every step rounds once, a sum of H squares log2(H) + 8 deep at the least and
    H / 64 + 10 at the most (halved by the root); the sigmoid is good to 4 ulps."""
    H = x.shape[-1]
    deep = (H / 64 + 10) / 2 + 6
    h = x.double()
    if p is not None:
        h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * p.double()
    if gate is not None:
        h = h * (torch.sigmoid(gate.double()) if sigmoid else gate.double())
    off = ULP32 * h.abs() * ((deep if p is not None else 0) + 6)
    z = residual_scale * r.double() + scale * h
    off = abs(scale) * off + ULP32 * ((scale * h).abs() + (residual_scale * r.double()).abs() + z.abs())
    y = off_y = None
    if w is not None:
        rstd = 1 / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)
        y = z * rstd * w.double()
        # d y: the value's own error, and the norm's by the root mean square of the row's errors (Cauchy's inequality)
        rel = (off * off).mean(-1, keepdim=True).sqrt() * rstd
        off_y = (off * rstd * w.double().abs()) + y.abs() * (rel + deep * ULP32)
    return z, off, y, off_y


def _check(got, want, dtype):
    z, off, y, off_y = want
    assert ((got.residual.double() - z).abs() <= 1.01 * (off + half_step(dtype, z))).all()
    if got.normed is not None:
        assert ((got.normed.double() - y).abs() <= 1.01 * (off_y + half_step(dtype, y))).all()


def _check_codes(got, form, y, off_y):
    """Scales to the maximum's error; a code's value is within half a step (int8 groups: a step, towards zero) of y, given y's error."""
    s = got.scale.double()
    v = y.unflatten(-1, (s.shape[-1], -1))
    off = off_y.unflatten(-1, (s.shape[-1], -1))
    most = 448.0 if form[0] == fp8_ref.FP8 else 127.0
    top = v.abs().amax(-1).clamp(min=1e-10)
    worst = off.amax(-1) + 3 * ULP32 * top
    assert ((s * most - top).abs() <= worst).all()
    q = got.q.double().unflatten(-1, (s.shape[-1], -1))
    slack = off + 6 * ULP32 * v.abs() + worst.unsqueeze(-1) * v.abs() / top.unsqueeze(-1)
    quotient, s = v / s.unsqueeze(-1), s.unsqueeze(-1)
    if form[0] == fp8_ref.FP8:
        step = 0.5 * fp8_ref.e4m3_step(quotient.abs() + slack / s)
        assert ((q - quotient).abs() <= step + slack / s).all()
    elif form[1] is None:
        assert ((q - quotient).abs() <= 0.5 + slack / s).all() and (q.abs() <= 127).all()
    else:
        low, high = quotient.abs() - 1 - slack / s, quotient.abs() + slack / s
        assert ((q.abs() >= low) & (q.abs() <= high)).all() and (q * quotient >= 0).all()


def _call(args, form, sigmoid=False, scale=1.0, residual_scale=1.0, eps=1e-6, **k):
    from lightop_amd.norm import rms_norm_block

    x, r, w, p, gate = args
    quant = form or (None, None)
    return rms_norm_block(x, r, w, post_weight=p, gate=gate, gate_activation="sigmoid" if sigmoid else None, scale=scale,
                          residual_scale=residual_scale, eps=eps, quant_dtype=quant[0], group_size=quant[1], **k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("M,H", [(1, 128), (1, 2048), (3, 256), (5, 7168), (70, 1024), (333, 4096), (769, 640), (1000, 5120), (2, 32768), (3, 65536)])
def test_sizes(dtype, form, M, H):
    print("[case] norm block", dtype, form, M, H, flush=True)
    options = [(None, True, False, 1.0, 1.0), ("token", True, True, 0.5, 1.0), ("channel", False, False, 1.0, 0.9), ("full", True, True, 2.0, -1.5),
               (None, False, False, -0.3, 1.0), ("token", False, False, 1.0, 0.0)]
    for i, (gate, post, sigmoid, scale, rs) in enumerate(options):
        args = _make(M, H, dtype, gate, post, i)
        want = _exact(*args, sigmoid, scale, rs, 1e-6)
        got = _call(args, form, sigmoid, scale, rs, return_normed=True)
        _check(got, want, dtype)
        if form is None:
            assert got.q is None and got.scale is None
        else:
            _check_codes(got, form, want[2], want[3])


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("M,H", [(2047, 2048), (2048, 2048), (2301, 1152), (3001, 128), (2050, 2176), (1100, 5248)])
def test_many_rows(form, M, H):
    print("[case] norm block", form, M, H, flush=True)
    for dtype, gate in ((torch.bfloat16, "channel"), (torch.float32, "token")):
        args = _make(M, H, dtype, gate, True)
        want = _exact(*args, True, 0.5, 1.0, 1e-6)
        got = _call(args, form, True, 0.5, return_normed=True)
        _check(got, want, dtype)
        if form is not None:
            _check_codes(got, form, want[2], want[3])


@pytest.mark.parametrize("H", [8, 24, 40, 520, 2056, 16392])
@pytest.mark.parametrize("form", [None, (torch.int8, None)], ids=str)
def test_odd_rows(H, form):
    for dtype in (torch.bfloat16, torch.float32):
        args = _make(7, H, dtype, "channel", True)
        want = _exact(*args, True, 1.0, 1.0, 1e-5)
        got = _call(args, form, True, eps=1e-5, return_normed=True)
        _check(got, want, dtype)
        if form:
            _check_codes(got, form, want[2], want[3])


@pytest.mark.parametrize("rows", [3, 2000])
def test_gates_of_every_layout(rows):
    B, T, H = 2, rows, 256
    g = torch.Generator(device="cuda").manual_seed(1)
    x, r, w = _normal(g, B, T, H), _normal(g, B, T, H), 1 + 0.1 * _normal(g, H)
    every = _normal(g, B, T, 2 * H)
    gates = [_normal(g, H), _normal(g, 1), _normal(g, B, 1, H), _normal(g, 1, T, H), _normal(g, T, 1), _normal(g, B, T, 1), _normal(g, B, 1, 1),
             every[..., :H], every[..., H:], every[..., ::2], every[..., 1:H + 1], every[:, :, :1], every[:, :1, H:], _normal(g, T, B, H).transpose(0, 1),
             _normal(g, H).to(torch.float32)[None, None].expand(B, T, H), _normal(g, B, T).unsqueeze(-1).expand(B, T, H), _normal(g, T, B).t().unsqueeze(-1)]
    for k, gate in enumerate(gates):
        for sigmoid in (False, True):
            got = _call((x, r, w, None, gate), None, sigmoid)
            want = _call((x, r, w, None, gate.expand(B, T, H).contiguous()), None, sigmoid)
            assert torch.equal(got.residual, want.residual) and torch.equal(got.normed, want.normed), k
            _check(got, _exact(x, r, w, None, gate, sigmoid, 1.0, 1.0, 1e-6), torch.float32)
    half = _call((x.bfloat16(), r.bfloat16(), w.bfloat16(), None, gates[2]), None)  # an fp32 gate beside 16-bit rows
    _check(half, _exact(x.bfloat16(), r.bfloat16(), w.bfloat16(), None, gates[2], False, 1.0, 1.0, 1e-6), torch.bfloat16)


@pytest.mark.parametrize("M", [3, 900])
def test_is_the_plain_norm_where_nothing_is_added(M):
    """Without post_weight, gate and scales: bit for bit ``rms_norm_quant`` with a residual."""
    from lightop_amd.norm import rms_norm_quant

    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x, r, w, _, _ = args = _make(M, 1024, dtype, None, False)
        for form in FORMS[1:]:
            got = _call(args, form, return_normed=True)
            want = rms_norm_quant(x, w, 1e-6, residual=r, quant_dtype=form[0], group_size=form[1], return_normed=True)
            assert torch.equal(got.residual, want.residual) and torch.equal(got.normed, want.normed) and torch.equal(got.scale, want.scale)
            assert torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8))


def test_outputs_strides_and_overlaps(monkeypatch):
    from lightop_amd import _lib
    from lightop_amd.norm import rms_norm_block

    x, r, w, p, gate = args = _make(40, 256, torch.bfloat16, "token", True)
    want = _call(args, None)
    place = r.clone()
    got = rms_norm_block(x, place, w, post_weight=p, gate=gate, residual_out=place)
    assert got.residual is place and torch.equal(place, want.residual) and torch.equal(got.normed, want.normed)
    place = x.clone()
    got = rms_norm_block(place, r, w, post_weight=p, gate=gate, residual_out=place)
    assert torch.equal(place, want.residual) and torch.equal(got.normed, want.normed)
    wide = torch.full((42, 300), float("nan"), dtype=x.dtype, device="cuda")
    wide[1:41, 8:264] = x
    off = torch.zeros(40 * 256 + 1, dtype=x.dtype, device="cuda")[1:].view(40, 256).copy_(r)
    got = rms_norm_block(wide[1:41, 8:264], off, w, post_weight=p, gate=gate)
    assert torch.equal(got.residual, want.residual) and torch.equal(got.normed, want.normed)
    got = rms_norm_block(x, r, w, post_weight=p, gate=gate, residual_out=off)
    assert got.residual is off and torch.equal(off, want.residual)
    room = torch.full((42, 256), 7.0, dtype=x.dtype, device="cuda")
    got = rms_norm_block(x, r, w, post_weight=p, gate=gate, residual_out=room[1:41])
    assert torch.equal(room[1:41], want.residual) and (room[0] == 7).all() and (room[41] == 7).all()
    only = rms_norm_block(x, r, post_weight=p, gate=gate)
    assert torch.equal(only.residual, want.residual) and only.normed is None and only.q is None
    with monkeypatch.context() as m:
        m.setattr(_lib, "_host", _lib._NoHost())
        got = _call(args, FORMS[1], return_normed=True)
        assert torch.equal(got.normed, want.normed)
    assert torch.equal(_call(args, FORMS[1]).q, got.q)
    room[:40] = r
    for bad in (lambda: rms_norm_block(x, room[:40], w, residual_out=room[1:41]), lambda: rms_norm_block(room[1:41], r, w, residual_out=room[:40]),
                lambda: rms_norm_block(x, r, w, gate=room[:40], residual_out=room[:40])):
        with pytest.raises(RuntimeError, match="overlaps"):
            bad()
    empty = rms_norm_block(x[:0], r[:0], w, gate=gate[:0], quant_dtype=torch.int8)
    assert empty.q.shape == (0, 256) and empty.scale.shape == (0, 1) and empty.residual.shape == (0, 256)


def test_rows_of_zeros_infinities_and_nans():
    x, r, w, p, gate = _make(6, 512, torch.bfloat16, "token", True)
    x[1], r[1] = 0, 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    gate[4] = float("-inf")
    r[5, 3] = float("-inf")
    clean = _make(6, 512, torch.bfloat16, "token", True)
    for form in FORMS:
        got, want = (_call(t, form, True, return_normed=True) for t in ((x, r, w, p, gate), clean))
        assert torch.equal(got.residual[0], want.residual[0]) and torch.equal(got.normed[0], want.normed[0])
        assert (got.residual[1] == 0).all() and (got.normed[1] == 0).all()
        assert got.residual[2].isnan().all() and got.normed[2].isnan().all()  # the norm's sum is a NaN
        assert got.residual[3, 9].isnan()                                     # inf * 0
        assert torch.equal(got.residual[4], r[4])                             # a closed gate
        assert got.residual[5, 3] == float("-inf") and got.normed[5, 3].isnan() and (got.normed[5, 4:] == 0).all()
        if form:
            assert (got.q[1].float() == 0).all() and torch.equal(got.q[0].view(torch.uint8), want.q[0].view(torch.uint8))


def test_more_rows_than_a_launch_takes():
    M = (1 << 21) + 5
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r, w = _normal(g, M, 8).bfloat16(), _normal(g, M, 8).bfloat16(), _normal(g, 8).bfloat16()
    gate = _normal(g, M, 1).bfloat16()
    got = _call((x, r, w, None, gate), None)
    _check(got, _exact(x, r, w, None, gate, False, 1.0, 1.0, 1e-6), torch.bfloat16)


def test_offsets_past_32_bits():
    M, H = 70000, 65536
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.zeros(M, H, dtype=torch.bfloat16, device="cuda")
    x[-3:] = _normal(g, 3, H).bfloat16()
    r, w = x, (1 + 0.1 * _normal(g, H)).bfloat16()
    got = _call((x, r, w, None, x), None)
    assert (got.residual[:100] == 0).all()
    got = type(got)(got.residual[-3:], got.normed[-3:], None, None)
    _check(got, _exact(x[-3:], x[-3:], w, None, x[-3:], False, 1.0, 1.0, 1e-6), torch.bfloat16)


def test_streams_and_graphs():
    args = _make(300, 1024, torch.bfloat16, "channel", True)
    want = _call(args, FORMS[3], True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _call(args, FORMS[3], True)
    side.synchronize()
    assert torch.equal(got.residual, want.residual) and torch.equal(got.scale, want.scale)
    x, r = args[0].clone(), args[1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = _call((x, r) + args[2:], FORMS[3], True)
    for k in range(3):
        x.copy_(args[0] * (k + 1))
        graph.replay()
        eager = _call((x, r) + args[2:], FORMS[3], True)
        torch.cuda.synchronize()
        assert torch.equal(made.residual, eager.residual) and torch.equal(made.scale, eager.scale)
        assert torch.equal(made.q.view(torch.uint8), eager.q.view(torch.uint8))


def test_refusals():
    from lightop_amd.norm import rms_norm_block

    x, r, w, p, gate = _make(4, 256, torch.bfloat16, "token", True)
    bad = [lambda: rms_norm_block(x, r.float(), w), lambda: rms_norm_block(x, r[:3], w), lambda: rms_norm_block(x, r, w[:128]), lambda: rms_norm_block(x, r, w.half()),
           lambda: rms_norm_block(x, r, w, post_weight=p.double()), lambda: rms_norm_block(x, r, w, gate=gate[:3]), lambda: rms_norm_block(x, r, w, gate=gate.half()),
           lambda: rms_norm_block(x, r, w, gate=x[:, :2]), lambda: rms_norm_block(x, r, w, gate=gate[None]), lambda: rms_norm_block(x, r, None, return_normed=True),
           lambda: rms_norm_block(x, r, None, quant_dtype=torch.int8), lambda: rms_norm_block(x, r, w, quant_dtype=torch.float8_e4m3fn),
           lambda: rms_norm_block(x, r, w, group_size=128), lambda: rms_norm_block(x[:, :100], r[:, :100], w[:100]), lambda: rms_norm_block(x, r, w, eps=-1.0),
           lambda: rms_norm_block(x, r, w, residual_out=r.float()), lambda: rms_norm_block(x, r, w, residual_out=torch.empty(256, 4, dtype=x.dtype, device="cuda").t()),
           lambda: rms_norm_block(x, r.cpu(), w), lambda: rms_norm_block(x.int(), r.int(), w)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        rms_norm_block(x, r, w, gate=gate, gate_activation="tanh")
