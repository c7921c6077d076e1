"""Smallest and largest sizes of the product and the adjusted logits that their documentation allows and a test can hold."""
import pytest

from test_linear_gpu import _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("tokens,columns,outputs", [(1, 1, 1), (1, 3, 2), (2, 1, 1), (40, 1, 1), (70, 7, 3), (300, 1, 9), (65, 15, 1), (33, 17, 8),
                                                    (100_003, 72, 136), (70_001, 16, 9), (5, 100_000, 24), (40, 70_001, 130), (200, 50_008, 264)])
def test_products_at_the_edges(cuda, lily, kind, tokens, columns, outputs):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(tokens + columns + outputs)
    scratch = lily.SamplerScratch(64, max_rows=1, max_history=0)
    a, w, kw = _inputs(torch, g, tokens, columns, outputs, kind)
    for out_type in (torch.bfloat16, torch.float32):
        out = torch.full((tokens + 2, outputs), 7.0, dtype=out_type, device="cuda")
        residual = torch.randn((tokens, outputs), generator=g, device="cuda").to(out_type)
        scratch.linear(a, w, out[1:-1], residual=residual, **kw)
        _check(torch, out[1:-1], a, w, kw, residual=residual)
        assert (out[0] == 7).all() and (out[-1] == 7).all()
    assert scratch.status() == lily.OK


@pytest.mark.parametrize("rows,bf16", [(1, False), (3, True), (9, False)])
def test_the_largest_vocabulary(cuda, lily, rows, bf16):
    """Rows of 2^24 ids, whole rows and a part at the end of the ids that masks can name: bit for bit in binary32."""
    torch = cuda
    vocab = 1 << 24
    g = torch.Generator(device="cuda").manual_seed(rows)
    scratch = lily.SamplerScratch(vocab, max_rows=rows, max_history=40_000, max_list=32)
    for first in (0, 2 ** 31 - 1 - vocab):
        logits = torch.randn((rows, vocab), generator=g, device="cuda")
        logits = logits.bfloat16() if bf16 else logits
        ids = torch.randperm(vocab, generator=g, device="cuda")[:30_000].int()
        history = (ids.repeat(rows, 1) + first).contiguous()
        biased, banned = ids[:16], ids[-16:]
        values = torch.randn((rows, 16), generator=g, device="cuda")
        full = lambda n: torch.full((rows,), n, dtype=torch.int32, device="cuda")
        kw = dict(history_ids=history, history_len=full(30_000), bias_ids=(biased + first).repeat(rows, 1), bias_vals=values,
                  bias_len=full(16), ban_ids=(banned + first).repeat(rows, 1), ban_len=full(16))
        mask = None
        if first == 0:
            mask = torch.randint(-2 ** 31, 2 ** 31, (1, vocab // 32), generator=g, device="cuda").int()
            kw.update(mask=mask, mask_rows=full(0))
        want = logits.float().clone()
        want[:, biased.long()] += values
        l = want[:, ids.long()]
        # (A quotient in binary64, rounded once more, is binary32's: 53 bits are more than twice 24 and two.)
        l = torch.where(l > 0, (l.double() / 1.25).float(), l * 1.25) - (0.5 + 0.25)
        want[:, ids.long()] = l
        want[:, banned.long()] = float("-inf")
        if mask is not None:
            bits = (mask.view(-1, 1) >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).bool().view(-1)
            want[:, ~bits] = float("-inf")
        out = torch.empty((rows, vocab), device="cuda")
        params = [lily.SamplingParams(repetition_penalty=1.25, presence_penalty=0.5, frequency_penalty=0.25)] * rows
        scratch.adjust_logits(logits, params, out, first_id=first, **kw)
        assert torch.equal(out, want), int((out != want).sum())
        if not bf16:
            scratch.adjust_logits(logits, params, first_id=first, **kw)
            assert torch.equal(logits, want)
    assert scratch.status() == lily.OK
