"""Products under wait limits shorter than a copy's way: a block that gives up stays until what it asked for
has landed. Such a call reports the wait or is right, and the next one finds everything as it should be."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("limit", [1, 300, 2_000, 20_000])
@pytest.mark.parametrize("tokens,columns,outputs", [(1, 4096, 300), (20, 2048, 40_000), (30, 8192, 256), (64, 1024, 20_000),
                                                    (70, 4096, 200), (300, 512, 1024), (600, 4096, 2048)])
def test_short_limits(cuda, lily, limit, tokens, columns, outputs):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(tokens + outputs)
    scratch = lily.SamplerScratch(64, max_rows=1, max_history=0)
    a = torch.randn((tokens, columns), generator=g, device="cuda").bfloat16()
    w = (torch.randn((outputs, columns), generator=g, device="cuda") / columns ** 0.5).bfloat16()
    residual = torch.randn((tokens, outputs), generator=g, device="cuda").bfloat16()
    want, out = torch.empty_like(residual), torch.empty_like(residual)
    scratch.linear(a, w, want, residual=residual)
    assert scratch.status() == lily.OK
    for _ in range(10):
        scratch.set_wait_limit(limit)
        out.zero_()
        scratch.linear(a, w, out, residual=residual)
        said = scratch.status()
        assert said in (lily.OK, lily.ERR_TIMEOUT)
        assert said == lily.ERR_TIMEOUT or torch.equal(out, want)
        scratch.set_wait_limit(0)
        scratch.linear(a, w, out, residual=residual)
        assert scratch.status() == lily.OK and torch.equal(out, want)
