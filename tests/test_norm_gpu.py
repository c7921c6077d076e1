"""lily_add_rms_norm on the GPU against the formula in 64 bits.

What may differ: h = x + residual rounds once (2^-24 relative to h); the sum of squares is a thread's
chain of at most 32 terms and ten levels of pairs, so 42 roundings of 2^-24, halved by the root; the root,
the quotient and the three products are five more: less than 2^-18 relative to a value. Then the
rounding to out's type: half a step."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32_ERROR = 2.0 ** -18
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}


def _handle(lily):
    return lily.SamplerScratch(64, max_rows=1, max_history=0)


def _rows(torch, g, tokens, hidden, dtype, pitch=0, offset=0, scale=1.0):
    """[tokens, hidden] of the type, rows `pitch` apart (0: contiguous), the first `offset` elements into its
    buffer, and the buffer, poisoned around the rows."""
    ld = pitch or hidden
    buf = torch.full((offset + tokens * ld + 64,), float("nan"), dtype=dtype, device="cuda")
    view = buf[offset:offset + tokens * ld].view(tokens, ld)[:, :hidden]
    view.copy_(torch.randn((tokens, hidden), generator=g, device="cuda") * scale)
    return view, buf


def _exact(torch, x, residual, weight, eps, offset):
    h = x.double() + (residual.double() if residual is not None else 0.0)
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * (offset + weight.double())
    return h, y


def _check(torch, out, scales, h, y, summed=None):
    if out.dtype == torch.float8_e4m3fn:
        m = y.abs().amax(1).clamp_min(2.0 ** -64)
        assert ((scales.double() - m / 448).abs() <= 2 * F32_ERROR * m / 448).all()
        value = out.double() * scales.double()[:, None]
        # Half a step of e4m3 is 2^-4 of the value, 2^-10 of the scale among its subnormals.
        tol = y.abs() * (2.0 ** -4 + 4 * F32_ERROR) + (2.0 ** -10 * m / 448)[:, None]
        assert ((value - y).abs() <= tol).all()
        # No row wastes its codes: its largest value lies in the topmost step.
        assert (out.double().abs().amax(1)[m > 2.0 ** -60] == 448).all()
    else:
        half = HALF_STEP[str(out.dtype).split(".")[1]]
        assert ((out.double() - y).abs() <= y.abs() * (half + F32_ERROR) + 1e-40).all()
    if summed is not None:
        half = HALF_STEP[str(summed.dtype).split(".")[1]]
        assert ((summed.double() - h).abs() <= h.abs() * (half + 2.0 ** -23)).all()


@pytest.mark.parametrize("tokens,hidden", [(1, 1), (1, 2048), (3, 7), (2, 31), (5, 1000), (64, 4096), (300, 96), (7, 5001),
                                           (2, 8191), (3, 8192), (2, 16384), (2, 16385), (1, 32768), (400, 513)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_norm_equals_the_formula(cuda, lily, tokens, hidden, dtype):
    torch = cuda
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(tokens * 100_003 + hidden)
    scratch = _handle(lily)
    for out_type in (torch.float32, torch.bfloat16, torch.float8_e4m3fn):
        for with_residual in (True, False):
            for weight_type, offset in ((torch.bfloat16, 0.0), (torch.float32, 1.0)):
                x, _ = _rows(torch, g, tokens, hidden, dtype, scale=3.0)
                residual = _rows(torch, g, tokens, hidden, dtype)[0] if with_residual else None
                weight = (torch.randn(hidden, generator=g, device="cuda") * 0.5 + (1.0 - offset)).to(weight_type)
                summed = torch.empty_like(x) if with_residual else None
                out = torch.empty((tokens, hidden), dtype=out_type, device="cuda")
                scales = torch.empty(tokens, device="cuda") if out_type == torch.float8_e4m3fn else None
                scratch.add_rms_norm(x, weight, out, residual=residual, residual_out=summed, out_scales=scales, eps=1e-5,
                                     weight_offset=offset)
                h, y = _exact(torch, x, residual, weight, 1e-5, offset)
                _check(torch, out, scales, h, y, summed)
    assert scratch.status() == 0


@pytest.mark.parametrize("hidden,pitch,offset", [(512, 520, 0), (512, 513, 0), (512, 512, 1), (100, 137, 3), (4096, 4104, 8)])
def test_rows_of_any_pitch_and_alignment(cuda, lily, hidden, pitch, offset):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(pitch)
    scratch, tokens = _handle(lily), 9
    for dtype, out_type in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.float8_e4m3fn)):
        x, _ = _rows(torch, g, tokens, hidden, dtype, pitch, offset)
        residual, _ = _rows(torch, g, tokens, hidden, dtype, pitch + 1, offset)
        summed, summed_buf = _rows(torch, g, tokens, hidden, dtype, pitch, offset)
        weight = torch.randn(hidden + 1, generator=g, device="cuda")[1:]
        out_buf = torch.full((offset + tokens * pitch + 64,), 0x55, dtype=torch.uint8, device="cuda")
        if out_type == torch.bfloat16:
            out_buf = out_buf.repeat(2).view(torch.bfloat16)
        out = out_buf.view(out_type)[offset:offset + tokens * pitch].view(tokens, pitch)[:, :hidden]
        before = out_buf.clone()
        scales = torch.full((tokens + 2,), -7.0, device="cuda")
        kw = {"out_scales": scales[1:tokens + 1]} if out_type == torch.float8_e4m3fn else {}
        scratch.add_rms_norm(x, weight, out, residual=residual, residual_out=summed, **kw)
        h, y = _exact(torch, x, residual, weight, 1e-6, 0.0)
        _check(torch, out, kw.get("out_scales"), h, y, summed)
        # Nothing beside the rows was written.
        outside = torch.ones(out_buf.shape, dtype=torch.bool, device="cuda")
        outside[offset:offset + tokens * pitch].view(tokens, pitch)[:, :hidden] = False
        assert torch.equal(out_buf.view(torch.uint8 if out_type == torch.float8_e4m3fn else torch.int16)[outside],
                           before.view(torch.uint8 if out_type == torch.float8_e4m3fn else torch.int16)[outside])
        gaps = torch.ones(summed_buf.shape, dtype=torch.bool, device="cuda")
        gaps[offset:offset + tokens * pitch].view(tokens, pitch)[:, :hidden] = False
        assert torch.isnan(summed_buf[gaps]).all()
        assert scales[0] == -7.0 and scales[-1] == -7.0


def test_in_place(cuda, lily):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(5)
    scratch = _handle(lily)
    for tokens, hidden in ((3, 4096), (500, 2048), (2, 777)):
        x = torch.randn((tokens, hidden), generator=g, device="cuda").bfloat16()
        residual = torch.randn((tokens, hidden), generator=g, device="cuda").bfloat16()
        weight = torch.randn(hidden, generator=g, device="cuda").bfloat16()
        out, summed = torch.empty_like(x), torch.empty_like(x)
        scratch.add_rms_norm(x, weight, out, residual=residual, residual_out=summed)
        x2, residual2 = x.clone(), residual.clone()
        scratch.add_rms_norm(x2, weight, x2, residual=residual2, residual_out=residual2)
        assert torch.equal(x2, out) and torch.equal(residual2, summed)


def test_zeros_infinities_and_nan_stay_in_their_row(cuda, lily):
    torch = cuda
    scratch, hidden = _handle(lily), 1024
    x = torch.randn((5, hidden), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    x[0] = 0.0
    x[2, 17] = float("nan")
    x[3, 5] = float("inf")
    weight = torch.ones(hidden, device="cuda")
    for out_type in (torch.float32, torch.float8_e4m3fn):
        out = torch.empty((5, hidden), dtype=out_type, device="cuda")
        scales = torch.empty(5, device="cuda") if out_type == torch.float8_e4m3fn else None
        scratch.add_rms_norm(x, weight, out, out_scales=scales)
        f = out.float()
        assert (f[0] == 0).all()
        assert torch.isnan(f[2]).all() and torch.isnan(f[3, 5])
        if scales is None:
            assert (f[3].isnan() | (f[3] == 0)).all()
        else:
            assert scales[0] > 0 and torch.isnan(scales[2])
        keep = torch.tensor([1, 4], device="cuda")
        h, y = _exact(torch, x[keep], None, weight, 1e-6, 0.0)
        _check(torch, out.view(torch.uint8)[keep].view(out_type) if scales is not None else out[keep],
               None if scales is None else scales[keep], h, y)


def test_rows_do_not_depend_on_the_rows_beside_them(cuda, lily):
    """The same token alone, in a batch and in a long prompt: up to the order of the sum of squares."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(8)
    scratch = _handle(lily)
    x = torch.randn((2000, 4096), generator=g, device="cuda").bfloat16()
    weight = torch.randn(4096, generator=g, device="cuda").bfloat16()
    whole, again, few = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    scratch.add_rms_norm(x, weight, whole)
    scratch.add_rms_norm(x, weight, again)
    assert torch.equal(whole, again)
    scratch.add_rms_norm(x[500:503], weight, few[500:503])
    assert ((few[500:503].double() - whole[500:503].double()).abs() <= whole[500:503].double().abs() * 2.0 ** -7).all()


def test_captured_and_on_another_stream(cuda, lily):
    torch = cuda
    scratch = _handle(lily)
    x = torch.randn((16, 2048), device="cuda").bfloat16()
    weight = torch.ones(2048, device="cuda")
    out, want = torch.empty_like(x), torch.empty_like(x)
    scratch.add_rms_norm(x, weight, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        scratch.add_rms_norm(x, weight, out)
    x.mul_(2.0)
    scratch.add_rms_norm(x, weight, want)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    side = torch.cuda.Stream()
    out.zero_()
    side.wait_stream(torch.cuda.current_stream())
    scratch.add_rms_norm(x, weight, out, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


def test_refusals(cuda, lily):
    torch = cuda
    scratch = _handle(lily)
    x = torch.zeros((4, 64), device="cuda")
    w, out = torch.ones(64, device="cuda"), torch.zeros((4, 64), device="cuda")
    codes = torch.zeros((4, 64), dtype=torch.float8_e4m3fn, device="cuda")
    for kw in (dict(x=x.cpu()), dict(weight=w[:63]), dict(out=out[:3]), dict(x=x.half()), dict(residual=x.bfloat16()),
               dict(out=codes), dict(out_scales=torch.zeros(4, device="cuda")), dict(eps=-1.0), dict(eps=float("nan")),
               dict(weight_offset=float("inf")), dict(residual_out=x[:, :32]), dict(x=x.t()), dict(x=x[:0]),
               dict(out=codes, out_scales=torch.zeros(3, device="cuda")), dict(out=out, residual_out=out),
               dict(x=torch.zeros((1, 40000), device="cuda"))):
        call = {**dict(x=x, weight=w, out=out), **kw}
        with pytest.raises(lily.LilyError) as e:
            scratch.add_rms_norm(call.pop("x"), call.pop("weight"), call.pop("out"), **call)
        assert e.value.code in (lily.ERR_ARG, lily.ERR_CAPACITY), kw
    scratch.inject_fault(3)
    with pytest.raises(lily.LilyError) as e:
        scratch.add_rms_norm(x, w, out)
    assert e.value.code == lily.ERR_FAULT
    scratch.clear_fault()
    scratch.add_rms_norm(x, w, out)
    assert scratch.status() == lily.OK


@pytest.mark.parametrize("hidden,pitch", [(1000, 2 ** 31 + 8), (1001, 2 ** 31 + 3)])
def test_rows_beyond_32_bits(cuda, lily, hidden, pitch):
    """Rows more than 2^32 bytes apart, the sum in place: as rows that follow one another."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(hidden)
    scratch = lily.SamplerScratch(64, max_rows=1, max_history=0)
    x = torch.randn((3, hidden), generator=g, device="cuda").bfloat16()
    residual = torch.randn((3, hidden), generator=g, device="cuda").bfloat16()
    weight = torch.randn(hidden, generator=g, device="cuda")
    want, total = torch.empty_like(x), torch.empty_like(x)
    scratch.add_rms_norm(x, weight, want, residual=residual, residual_out=total)
    buffer = torch.empty(2 * pitch + hidden, dtype=torch.bfloat16, device="cuda")
    far = buffer.as_strided((3, hidden), (pitch, 1)).copy_(residual)
    out = torch.empty_like(x)
    scratch.add_rms_norm(x, weight, out, residual=far, residual_out=far)
    assert torch.equal(out, want) and torch.equal(far, total)
