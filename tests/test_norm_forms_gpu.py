"""lily_add_rms_norm in the forms that a call's sizes lead to: a warp per short row with one, two and four vectors a
lane, blocks with one to eight, rows on and off the boundaries, each in both types, with and without a residual; sums
and outs in place, also crosswise.

The bound of test_norm_gpu, for every form: a thread's chain is at most 64 terms (eight vectors), and ten levels of
pairs follow: 74 roundings of 2^-24, halved by the root; with the root, the quotients and the products below 2^-18."""
import pytest

from test_norm_gpu import _check, _exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,hidden", [(400, 8), (333, 256), (400, 264), (400, 512), (301, 520), (400, 1024), (333, 1032), (297, 2048),
                                           (310, 4096), (300, 8192), (299, 16384), (2, 1024), (2, 4096), (2, 8200), (2, 16392), (1, 32760),
                                           (2, 32761)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_every_form(cuda, lily, tokens, hidden, dtype):
    torch = cuda
    dtype = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(tokens * 31 + hidden)
    scratch = lily.SamplerScratch(64, max_rows=1, max_history=0)
    rows = lambda pad, t=dtype: torch.randn((tokens, hidden + pad), generator=g, device="cuda").to(t)[:, :hidden]
    for pad in (0, 3):
        for out_type in (torch.float32, torch.bfloat16, torch.float8_e4m3fn):
            for with_residual in (True, False):
                x, residual = rows(pad), rows(pad) if with_residual else None
                weight = rows(0)[0].contiguous()
                summed = torch.full((tokens, hidden + pad), 7.0, dtype=dtype, device="cuda")
                out = torch.full((tokens, hidden + pad), 7.0, device="cuda").to(out_type)
                scales = torch.empty(tokens, device="cuda") if out_type == torch.float8_e4m3fn else None
                scratch.add_rms_norm(x, weight, out[:, :hidden], residual=residual, residual_out=summed[:, :hidden], out_scales=scales,
                                     eps=1e-5)
                h, y = _exact(torch, x, residual, weight, 1e-5, 0.0)
                _check(torch, out[:, :hidden], scales, h, y, summed[:, :hidden])
                assert (out[:, hidden:].float() == 7).all() and (summed[:, hidden:] == 7).all()
    assert scratch.status() == lily.OK


@pytest.mark.parametrize("tokens,hidden", [(3, 2048), (400, 512), (400, 1000), (2, 777), (300, 5001), (2, 16384), (500, 8192)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_in_place_crosswise(cuda, lily, tokens, hidden, dtype):
    """out over the residual and the sum over x; out over x and the sum elsewhere; and the other way round."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(hidden)
    scratch = lily.SamplerScratch(64, max_rows=1, max_history=0)
    x, residual = (torch.randn((tokens, hidden), generator=g, device="cuda").to(getattr(torch, dtype)) for _ in range(2))
    weight = torch.randn(hidden, generator=g, device="cuda")
    out, summed = torch.empty_like(x), torch.empty_like(x)
    scratch.add_rms_norm(x, weight, out, residual=residual, residual_out=summed)
    for where in ((1, 0), (0, 1), (0, None), (1, None), (None, 0), (None, 1)):
        mine = [x.clone(), residual.clone()]
        to_out, to_sum = (torch.empty_like(x) if w is None else mine[w] for w in where)
        scratch.add_rms_norm(mine[0], weight, to_out, residual=mine[1], residual_out=to_sum)
        assert torch.equal(to_out, out) and torch.equal(to_sum, summed), where
    assert scratch.status() == lily.OK
