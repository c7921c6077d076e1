"""lily_linear on the GPU against the formula in 64 bits.

What may differ: the multiplier sums 16 (bf16) or 32 (e4m3) products and the running sum per step, to a few
units of the last of binary32's 24 bits: with S = sum |a w| at most 2^-22 S a step, so (steps + 8) * 2^-22 * S,
the shares' sums included. The epilogue's roundings and its exp, erf and tanh are below 2^-20 of the
values they take part in; the activations' slopes below 1.2. Then the rounding to out's type: half a step."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}


def _handle(lily):
    return lily.SamplerScratch(64, max_rows=1, max_history=0)


def _act(torch, y, act):
    if act == "relu":
        return y.clamp_min(0)
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu":
        return 0.5 * y * torch.erfc(-y * 0.5 ** 0.5)
    if act == "gelu_tanh":
        return y * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (y + 0.044715 * y ** 3))
    return y


def _inputs(torch, g, tokens, columns, outputs, kind, pitch=0):
    ld = (columns + 15) // 16 * 16 + pitch
    a = torch.randn((tokens, ld), generator=g, device="cuda")
    w = torch.randn((outputs, ld), generator=g, device="cuda") / columns ** 0.5
    kw = {}
    if kind == "e4m3":
        scales = []
        for m in (a, w):
            s = m.abs().amax(1) / 448 + 1e-20
            m.div_(s[:, None])
            scales.append(s)
        a, w = a.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
        kw = dict(a_scales=scales[0], weight_scales=scales[1])
    else:
        a, w = a.bfloat16(), w.bfloat16()
    return a[:, :columns], w[:, :columns], kw


def _check(torch, out, a, w, kw, bias=None, act="none", residual=None):
    ad, wd = a.double(), w.double()
    if "a_scales" in kw:
        ad, wd = ad * kw["a_scales"].double()[:, None], wd * kw["weight_scales"].double()[:, None]
    y, s = ad @ wd.t(), ad.abs() @ wd.abs().t()
    steps = a.shape[1] / (32 if "a_scales" in kw else 16)
    tol = (steps + 8) * 2.0 ** -22 * s
    if bias is not None:
        y = y + bias.double()
    pre = y
    y = _act(torch, y, act)
    tol = 1.2 * tol + 2.0 ** -20 * (pre.abs() + y.abs())
    if residual is not None:
        y = y + residual.double()
        tol = tol + 2.0 ** -24 * y.abs()
    tol = tol + (y.abs() + tol) * HALF_STEP[str(out.dtype).split(".")[1]] + 1e-38
    off = (out.double() - y).abs()
    assert (off <= tol).all(), (off - tol).max()


SIZES = [(1, 2048, 2048), (1, 16, 1), (1, 8, 130), (2, 100, 300), (7, 1000, 129), (16, 4096, 512), (17, 520, 257),
         (24, 4096, 4096), (32, 64, 128), (33, 192, 1000), (64, 2048, 777), (65, 512, 384), (128, 1024, 1024),
         (129, 320, 640), (200, 2048, 1000), (257, 640, 515), (512, 1024, 2048), (700, 96, 4096), (2049, 512, 1025),
         (150, 4096, 300), (300, 2064, 520), (513, 4096, 513), (1024, 2048, 1024), (190, 8192, 2050),
         (37, 256, 50257), (5, 128, 38001), (64, 1024, 11000), (16, 72, 40003), (30, 640, 21001)]


@pytest.mark.parametrize("tokens,columns,outputs", SIZES)
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_product_equals_the_formula(cuda, lily, tokens, columns, outputs, kind):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(tokens * 7 + columns * 3 + outputs)
    scratch = _handle(lily)
    a, w, kw = _inputs(torch, g, tokens, columns, outputs, kind)
    for out_type in (torch.float32, torch.bfloat16):
        out = torch.full((tokens + 2, outputs), 7.0, dtype=out_type, device="cuda")
        scratch.linear(a, w, out[1:tokens + 1], **kw)
        _check(torch, out[1:tokens + 1], a, w, kw)
        assert (out[0] == 7).all() and (out[-1] == 7).all()
    assert scratch.status() == 0


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("tokens,columns,outputs", [(1, 1024, 2048), (9, 264, 333), (100, 512, 512), (600, 256, 1030)])
def test_epilogue(cuda, lily, act, tokens, columns, outputs):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(tokens)
    scratch = _handle(lily)
    for kind, out_type, bias_type in (("bf16", torch.bfloat16, torch.bfloat16), ("e4m3", torch.float32, torch.float32),
                                      ("bf16", torch.float32, torch.bfloat16), ("e4m3", torch.bfloat16, torch.float32)):
        a, w, kw = _inputs(torch, g, tokens, columns, outputs, kind)
        bias = torch.randn(outputs, generator=g, device="cuda").to(bias_type)
        residual = torch.randn((tokens, outputs + 3), generator=g, device="cuda").to(out_type)[:, :outputs]
        out = torch.full((tokens, outputs + 5), 3.0, dtype=out_type, device="cuda")
        scratch.linear(a, w, out[:, :outputs], bias=bias, activation=act, residual=residual, **kw)
        _check(torch, out[:, :outputs], a, w, kw, bias, act, residual)
        assert (out[:, outputs:] == 3.0).all()
        # In place: the residual's buffer becomes out.
        mine = residual.clone()
        scratch.linear(a, w, mine, bias=bias, activation=act, residual=mine, **kw)
        assert torch.equal(mine, out[:, :outputs])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("tokens,columns,outputs", [(129, 128, 9480), (200, 72, 9600), (301, 512, 520), (385, 4096, 4096),
                                                    (600, 256, 1032), (1030, 1024, 256), (2500, 64, 1224), (300, 4096, 512),
                                                    (333, 128, 1003), (450, 64, 9481)])
def test_many_tokens_with_rows_on_boundaries(cuda, lily, kind, tokens, columns, outputs):
    """bf16 outs and residuals whose rows start on 16-byte boundaries: contiguous, as a part of wider rows, in
    place; tiles that end inside the tokens and the outputs leave what lies behind them."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(tokens + outputs)
    scratch = _handle(lily)
    a, w, kw = _inputs(torch, g, tokens, columns, outputs, kind)
    pitch = (outputs + 7) // 8 * 8
    for act, bias_type, wide, with_residual in (("none", None, 0, False), ("silu", torch.float32, 8, True),
                                                ("gelu", torch.bfloat16, 40, True), ("relu", None, 0, True)):
        bias = None if bias_type is None else torch.randn(outputs, generator=g, device="cuda").to(bias_type)
        residual = None
        if with_residual:
            residual = torch.randn((tokens, pitch + 2 * wide), generator=g, device="cuda").bfloat16()[:, wide:wide + outputs]
        out = torch.full((tokens + 2, pitch + 2 * wide), 3.0, dtype=torch.bfloat16, device="cuda")
        mine = out[1:-1, wide:wide + outputs]
        scratch.linear(a, w, mine, bias=bias, activation=act, residual=residual, **kw)
        _check(torch, mine, a, w, kw, bias, act, residual)
        assert (out[0] == 3).all() and (out[-1] == 3).all()
        assert (out[:, :wide] == 3).all() and (out[:, wide + outputs:] == 3).all()
        if residual is not None:
            place = torch.full_like(out, 3.0)
            mine2 = place[1:-1, wide:wide + outputs]
            mine2.copy_(residual)
            scratch.linear(a, w, mine2, bias=bias, activation=act, residual=mine2, **kw)
            assert torch.equal(place, out)
    assert scratch.status() == lily.OK


def test_rows_on_boundaries_and_off_them_give_the_same(cuda, lily):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(21)
    scratch = _handle(lily)
    a, w, kw = _inputs(torch, g, 700, 512, 1024, "bf16")
    residual = torch.randn((700, 1024), generator=g, device="cuda").bfloat16()
    out = torch.empty((700, 1024), dtype=torch.bfloat16, device="cuda")
    odd = torch.empty((700, 1025), dtype=torch.bfloat16, device="cuda")[:, 1:]
    odd_residual = torch.empty((700, 1027), dtype=torch.bfloat16, device="cuda")[:, 2:1026].copy_(residual)
    for act in ("none", "silu", "gelu", "gelu_tanh"):
        scratch.linear(a, w, out, activation=act, residual=residual)
        scratch.linear(a, w, odd, activation=act, residual=odd_residual)
        assert torch.equal(out, odd)


def test_lost_copy_among_shares(cuda, lily):
    """Few tiles of long columns, which several blocks share: one of them gives up, all of them end. And many
    tiles in turn."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(23)
    scratch = _handle(lily)
    for tokens, outputs in ((70, 200), (300, 256), (300, 1024), (500, 2048), (30, 40000), (64, 11000)):
        a, w, kw = _inputs(torch, g, tokens, 4096, outputs, "bf16")
        out = torch.empty((tokens, outputs), device="cuda")
        for stage in (0, 6):
            scratch.set_wait_limit(20_000_000)
            scratch.inject_lost_copy(stage)
            scratch.linear(a, w, out)
            assert scratch.status() == lily.ERR_TIMEOUT
            scratch.set_wait_limit(0)
            scratch.linear(a, w, out)
            assert scratch.status() == lily.OK
            _check(torch, out, a, w, kw)


def test_lost_copy_with_a_residual(cuda, lily):
    """The residual's copies are under way when the wait runs out; the next call is right."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(22)
    scratch = _handle(lily)
    a, w, kw = _inputs(torch, g, 900, 1024, 2048, "bf16")
    residual = torch.randn((900, 2048), generator=g, device="cuda").bfloat16()
    out = torch.empty_like(residual)
    for stage in (0, 3, 15):
        scratch.set_wait_limit(20_000_000)
        scratch.inject_lost_copy(stage)
        scratch.linear(a, w, out, residual=residual)
        assert scratch.status() == lily.ERR_TIMEOUT
        scratch.set_wait_limit(0)
        scratch.linear(a, w, out, residual=residual)
        assert scratch.status() == lily.OK
        _check(torch, out, a, w, kw, residual=residual)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_exact_where_the_sums_are(cuda, lily, kind):
    """Small integers: every partial sum is exact in binary32, in any order and any shares."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(3)
    scratch = _handle(lily)
    for tokens, columns, outputs in ((1, 4096, 1000), (20, 2048, 300), (50, 1024, 2000), (130, 4096, 260), (1030, 1040, 2055)):
        a = torch.randint(-4, 5, (tokens, columns), generator=g, device="cuda").float()
        w = torch.randint(-4, 5, (outputs, columns), generator=g, device="cuda").float()
        want = (a.double() @ w.double().t()).float()
        kw = {}
        t = torch.bfloat16
        if kind == "e4m3":
            t = torch.float8_e4m3fn
            kw = dict(a_scales=torch.ones(tokens, device="cuda"), weight_scales=torch.ones(outputs, device="cuda"))
        out = torch.empty((tokens, outputs), device="cuda")
        scratch.linear(a.to(t), w.to(t), out, **kw)
        assert torch.equal(out, want), (tokens, columns, outputs)


def test_padding_between_rows_is_not_read(cuda, lily):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(4)
    scratch = _handle(lily)
    for tokens in (5, 300):
        for columns in (72, 1000, 65):
            a, w, kw = _inputs(torch, g, tokens, columns, 200, "bf16", pitch=64)
            for m in (a, w):
                m.as_strided((m.shape[0], m.stride(0) - columns), m.stride(), m.storage_offset() + columns).fill_(float("nan"))
            out = torch.empty((tokens, 200), device="cuda")
            scratch.linear(a, w, out)
            _check(torch, out, a, w, kw)


def test_nan_and_infinity_stay_in_their_token(cuda, lily):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(9)
    scratch = _handle(lily)
    for tokens in (4, 400):
        a, w, kw = _inputs(torch, g, tokens, 512, 256, "bf16")
        a[1, 3] = float("nan")
        a[2, 8] = float("inf")
        for act in ("none", "relu", "silu", "gelu", "gelu_tanh"):
            out = torch.empty((tokens, 256), device="cuda")
            scratch.linear(a, w, out, activation=act)
            assert torch.isnan(out[1]).all()
            assert not torch.isfinite(out[2][w[:, 8] > 0]).any()
            rest = torch.tensor([0, 3], device="cuda")
            _check(torch, out[rest], a[rest], w, kw, act=act)


def test_same_results_again_and_beside_other_tokens(cuda, lily):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(10)
    scratch = _handle(lily)
    a, w, kw = _inputs(torch, g, 64, 4096, 1024, "bf16")
    out, again = torch.empty((64, 1024), device="cuda"), torch.empty((64, 1024), device="cuda")
    scratch.linear(a, w, out)
    for _ in range(3):
        scratch.linear(a, w, again)
        assert torch.equal(out, again)
    scratch.linear(a[:40], w, again[:40])
    assert torch.equal(out[:40], again[:40])


def test_captured_and_two_streams_at_once(cuda, lily):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(11)
    scratch = _handle(lily)
    cases = []
    for tokens in (1, 40, 600):
        a, w, kw = _inputs(torch, g, tokens, 1024, 1024, "bf16")
        want = torch.empty((tokens, 1024), device="cuda")
        scratch.linear(a, w, want)
        cases.append((a, w, want))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a, w, want in cases:
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want)
        with torch.cuda.graph(graph):
            scratch.linear(a, w, out)
        graphs.append(graph)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):  # captured calls of one handle, side by side
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for out, (_, _, want) in zip(outs, cases):
        assert torch.equal(out, want)
    assert scratch.status() == 0


def test_a_wait_that_runs_out_is_reported(cuda, lily):
    """A copy that is never asked for: the launch ends, the status says so, the handle stays usable."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(12)
    scratch = _handle(lily)
    for tokens in (1, 100, 600):
        a, w, kw = _inputs(torch, g, tokens, 2048, 2048, "bf16")
        out = torch.empty((tokens, 2048), device="cuda")
        scratch.set_wait_limit(20_000_000)
        scratch.inject_lost_copy(1)
        scratch.linear(a, w, out)
        assert scratch.status() == lily.ERR_TIMEOUT
        scratch.set_wait_limit(0)
        scratch.linear(a, w, out)
        assert scratch.status() == lily.OK
        _check(torch, out, a, w, kw)


@pytest.mark.parametrize("tokens,pitch", [(3, 2 ** 31 + 8), (70, 2 ** 26), (70, 2 ** 26 + 1)])
def test_offsets_beyond_32_bits(cuda, lily, tokens, pitch):
    """Rows of a and out that lie more than 2^32 bytes apart in all; the residual is out itself."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(24)
    scratch = _handle(lily)
    buffer = torch.empty((tokens - 1) * pitch + 4096, dtype=torch.bfloat16, device="cuda")
    a, w, kw = _inputs(torch, g, tokens, 256, 520, "bf16")
    if pitch % 8 == 0:
        a = buffer.as_strided((tokens, 256), (pitch, 1), 1024).copy_(a)
    out = buffer.as_strided((tokens, 520), (pitch, 1))
    residual = torch.randn((tokens, 520), generator=g, device="cuda").bfloat16()
    out.copy_(residual)
    scratch.linear(a, w, out, residual=out)
    _check(torch, out, a, w, kw, residual=residual)


def test_refusals(cuda, lily):
    torch = cuda
    scratch = _handle(lily)
    bf, f8 = torch.bfloat16, torch.float8_e4m3fn
    a, w, out = (torch.zeros((4, 64), dtype=bf, device="cuda"), torch.zeros((32, 64), dtype=bf, device="cuda"),
                 torch.zeros((4, 32), device="cuda"))
    ones = lambda n: torch.ones(n, device="cuda")
    for kw in (dict(a=a.float()), dict(weight=w.to(f8)), dict(a=a.to(f8), weight=w.to(f8)), dict(a_scales=ones(4)),
               dict(a_scales=ones(4), weight_scales=ones(32)), dict(weight=w[:, :32]), dict(out=out[:, :31]),
               dict(out=out.half()), dict(bias=ones(31)), dict(residual=out.bfloat16()), dict(residual=out[:3]),
               dict(activation="tanh"), dict(a=a.cpu()), dict(a=a[:0]), dict(a=a.t()),
               dict(a=torch.zeros((4, 65), dtype=bf, device="cuda")[:, :64]),
               dict(a=torch.zeros(4 * 64 + 1, dtype=bf, device="cuda")[1:].view(4, 64)),
               dict(a=a.to(f8), weight=w.to(f8), a_scales=ones(3), weight_scales=ones(32))):
        call = {**dict(a=a, weight=w, out=out), **kw}
        with pytest.raises(lily.LilyError) as e:
            scratch.linear(call.pop("a"), call.pop("weight"), call.pop("out"), **call)
        assert e.value.code in (lily.ERR_ARG, lily.ERR_CAPACITY), kw
    scratch.linear(a, w, out)
    assert scratch.status() == lily.OK
