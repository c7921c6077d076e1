"""lily_add_rms_norm's 8-bit codes are those of the y that it writes in 32 bits, bit for bit: scale = m / 448,
code = e4m3(y * (448 / m)) with m = max(|y|, 2^-64), each step one rounding to binary32. And y itself against the
header's order of products."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _codes(torch, y):
    """On the host, quotients as IEEE has them (a tensor over a number is a product with its reciprocal there on the GPU)."""
    y = y.cpu().numpy()
    m = np.maximum(np.abs(y).max(1, keepdims=True), np.float32(2.0 ** -64))
    codes = torch.from_numpy(y * (np.float32(448.0) / m)).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.cuda(), torch.from_numpy((m / np.float32(448.0)).reshape(-1)).cuda()


@pytest.mark.parametrize("tokens,hidden", [(1, 2048), (64, 4096), (5, 1001), (400, 264), (400, 512), (333, 1024), (700, 4096),
                                           (310, 8192), (3, 16384), (2, 32768)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_codes_are_those_of_the_wide_values(cuda, lily, tokens, hidden, dtype):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(tokens * 3 + hidden)
    scratch = lily.SamplerScratch(64, max_rows=1, max_history=0)
    dtype = getattr(torch, dtype)
    for loud, eps in ((1.0, 1e-6), (2.0 ** -40, 0.0), (30.0, 1e-5)):
        for pad in (0, 8, 1):  # (rows on the 16-byte boundaries, and off them)
            x = torch.randn((tokens, hidden + pad), generator=g, device="cuda").mul(loud).to(dtype)[:, :hidden]
            residual = torch.randn((tokens, hidden + pad), generator=g, device="cuda").mul(loud).to(dtype)[:, :hidden]
            weight = (1.0 + 0.3 * torch.randn(hidden, generator=g, device="cuda")).bfloat16()
            # The same pitch in elements for all of them: one deal of the rows, one order of the sum.
            wide = torch.empty((tokens, hidden + pad), device="cuda")[:, :hidden]
            codes = torch.empty((tokens, hidden + pad), dtype=torch.float8_e4m3fn, device="cuda")[:, :hidden]
            scales = torch.empty(tokens, device="cuda")
            scratch.add_rms_norm(x, weight, wide, residual=residual, eps=eps)
            scratch.add_rms_norm(x, weight, codes, residual=residual, out_scales=scales, eps=eps)
            want, want_scales = _codes(torch, wide)
            assert torch.equal(scales, want_scales)
            assert torch.equal(codes.view(torch.uint8), want), int((codes.view(torch.uint8) != want).sum())
    assert scratch.status() == lily.OK


def test_the_smallest_tokens_have_codes(cuda, lily):
    """A token whose root mean square is near binary32's least normal, with weights that make its y tiny: the
    factor from h * weight to codes would pass binary32's range, y and 448 / m do not."""
    torch = cuda
    scratch = lily.SamplerScratch(64, max_rows=1, max_history=0)
    h = torch.full((2, 256), 2.0 ** -62, device="cuda")
    h[1, ::2] *= -0.5
    weight = torch.full((256,), 2.0 ** -62, device="cuda")
    wide, codes, scales = torch.empty_like(h), torch.empty(h.shape, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(2, device="cuda")
    scratch.add_rms_norm(h, weight, wide, eps=0.0)
    scratch.add_rms_norm(h, weight, codes, out_scales=scales, eps=0.0)
    want, want_scales = _codes(torch, wide)
    assert torch.equal(codes.view(torch.uint8), want) and torch.equal(scales, want_scales)
    # |y| is at most 2^-61, an eighth of 2^-58: by the floor of 2^-64 these are ordinary values.
    assert (codes.float().abs().amax(1) == 448).all()
