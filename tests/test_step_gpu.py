"""A decoding step from the last layer's output to the token, as an engine runs it: residual and norm
(lily_add_rms_norm), a gated block (lily_linear), the norm again, the head, the adjusted logits
(lily_adjust_logits) and the draw; whole, captured, and by vocabulary shards.

Each stage is compared with the formula in 64 bits of what the stage before it wrote, within that stage's
roundings: the norm's sum of squares and its root, 2^-20 of the value, then half a step of out's type (bf16
2^-8, e4m3 2^-4 of the value and, near zero, half its smallest step, 2^-10 codes). The product's bound is
the one of its own test."""
from __future__ import annotations

import pytest

from test_linear_gpu import _check as check_product

pytestmark = pytest.mark.gpu

EPS = 1e-6


class Block:
    """A layer's second half and the head, of a small model with odd sizes."""

    def __init__(self, torch, hidden=520, inner=1100, vocab=3204):
        g = torch.Generator(device="cuda").manual_seed(hidden + inner)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")
        self.hidden, self.inner, self.vocab = hidden, inner, vocab
        self.inner_ld = (inner + 15) // 16 * 16
        self.norm1, self.norm2 = 1 + 0.1 * rand(hidden), (0.1 * rand(hidden)).bfloat16()  # (the second: distance from 1)
        ld = (hidden + 15) // 16 * 16
        up = torch.zeros((inner, ld), device="cuda")
        up[:, :hidden] = rand(inner, hidden) / hidden ** 0.5
        self.up_scales = up.abs().amax(1) / 448
        self.up = (up / self.up_scales[:, None]).to(torch.float8_e4m3fn)[:, :hidden]
        self.bias = 0.1 * rand(inner)
        down = torch.zeros((hidden, self.inner_ld), device="cuda")
        down[:, :inner] = rand(hidden, inner) / inner ** 0.5
        self.down = down.bfloat16()[:, :inner]
        self.head = (rand(vocab, hidden) * 3 / hidden ** 0.5).bfloat16()
        self.ld = ld


class State:
    """What a step of so many tokens writes."""

    def __init__(self, torch, m, tokens, rows):
        e = lambda *s, dtype=torch.float32: torch.empty(s, dtype=dtype, device="cuda")
        self.x, self.residual = e(tokens, m.hidden, dtype=torch.bfloat16), e(tokens, m.hidden, dtype=torch.bfloat16)
        self.sum = torch.empty_like(self.x)
        self.y8, self.y8_scales = e(tokens, m.ld, dtype=torch.float8_e4m3fn)[:, :m.hidden], e(tokens)
        self.act = e(tokens, m.inner_ld, dtype=torch.bfloat16)[:, :m.inner]
        self.out = torch.empty_like(self.x)
        self.last = e(rows, m.hidden, dtype=torch.bfloat16)
        self.logits, self.adjusted = e(rows, m.vocab), e(rows, m.vocab)
        self.ids, self.status = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))

    def fill(self, torch, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (self.x, self.residual):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))


def _lists(torch, m, rows, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = lambda n: torch.randint(0, m.vocab, (rows, n), generator=g, device="cuda", dtype=torch.int32)
    full = lambda n: torch.full((rows,), n, dtype=torch.int32, device="cuda")
    lists = dict(history_ids=ids(700), history_len=full(700), bias_ids=ids(9), bias_len=full(9), ban_ids=ids(5), ban_len=full(5),
                 bias_vals=torch.randn((rows, 9), generator=g, device="cuda") * 3)
    lists["history_len"][0] = 0
    words = (m.vocab + 31) // 32
    mask = torch.randint(-2 ** 31, 2 ** 31, (2, words), generator=g, device="cuda").int()
    mask_rows = (torch.arange(rows, device="cuda") % 3 - 1).int()  # none, 0, 1, none, ...
    return lists, dict(mask=mask, mask_rows=mask_rows)


def _params(lily, rows):
    return [lily.SamplingParams(temperature=0.8, top_k=40, top_p=0.95, repetition_penalty=1.2, presence_penalty=0.3,
                                frequency_penalty=0.05, seed=r) for r in range(rows)]


def _step(lily, scratch, m, s, params, lists, masks, steps):
    scratch.add_rms_norm(s.x, m.norm1, s.y8, residual=s.residual, residual_out=s.sum, out_scales=s.y8_scales, eps=EPS)
    scratch.linear(s.y8, m.up, s.act, a_scales=s.y8_scales, weight_scales=m.up_scales, bias=m.bias, activation="silu")
    s.out.copy_(s.sum)
    scratch.linear(s.act, m.down, s.out, residual=s.out)
    rows = s.logits.shape[0]
    scratch.add_rms_norm(s.out[-rows:], m.norm2, s.last, eps=EPS, weight_offset=1.0)
    scratch.linear(s.last, m.head, s.logits)
    scratch.adjust_logits(s.logits, params, s.adjusted, out_status=s.status, **lists, **masks)
    scratch.sample_batch(s.adjusted, [lily.draft_params(p) for p in params], s.ids, steps=steps)


def _norm(h, weight, offset=0.0):
    h = h.double()
    return h / (h.square().mean(1, keepdim=True) + EPS).sqrt() * (offset + weight.double())


@pytest.mark.parametrize("tokens,rows", [(1, 1), (6, 6), (24, 24), (333, 7)])
def test_a_step_stage_by_stage(cuda, lily, tokens, rows):
    torch = cuda
    m, s = Block(torch), State(torch, Block(torch), tokens, rows)
    s.fill(torch, tokens)
    scratch = lily.SamplerScratch(m.vocab, max_rows=rows, max_history=1024)
    lists, masks = _lists(torch, m, rows, 5)
    params, steps = _params(lily, rows), list(range(rows))
    _step(lily, scratch, m, s, params, lists, masks, steps)
    assert scratch.status() == lily.OK and (s.status == 0).all()

    h = s.x.float() + s.residual.float()  # (rounded once, as the formula's sum is in binary32)
    assert torch.equal(s.sum, h.bfloat16())
    y = _norm(h, m.norm1)
    scales = s.y8_scales.double()[:, None]
    assert ((scales[:, 0] - y.abs().amax(1) / 448).abs() <= 2.0 ** -20 * scales[:, 0]).all()
    tol = y.abs() * (2.0 ** -4 + 2.0 ** -18) + scales * 2.0 ** -10 * 1.01
    assert ((s.y8.double() * scales - y).abs() <= tol).all()
    check_product(torch, s.act, s.y8, m.up, dict(a_scales=s.y8_scales, weight_scales=m.up_scales), m.bias, "silu")
    check_product(torch, s.out, s.act, m.down, {}, residual=s.sum)
    y = _norm(s.out[-rows:], m.norm2, 1.0)
    assert ((s.last.double() - y).abs() <= y.abs() * (2.0 ** -8 + 2.0 ** -18)).all()
    check_product(torch, s.logits, s.last, m.head, {})

    # The adjusted rows: what may not be drawn, and the draws against those with the lists built in.
    bits = (masks["mask"].view(2, -1, 1) >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).bool().reshape(2, -1)[:, :m.vocab]
    for r in range(rows):
        k = int(masks["mask_rows"][r])
        if k >= 0:
            assert (s.adjusted[r][~bits[k]] == float("-inf")).all()
            assert bits[k][int(s.ids[r])]
        assert int(s.ids[r]) not in lists["ban_ids"][r].tolist()
    again = torch.empty_like(s.ids)
    scratch.sample_batch(s.logits, params, again, steps=steps, **lists)
    free = masks["mask_rows"] < 0
    assert torch.equal(again[free], s.ids[free])


@pytest.mark.parametrize("tokens,rows", [(1, 1), (24, 24), (333, 7)])
def test_a_step_captured_and_replayed(cuda, lily, tokens, rows):
    torch = cuda
    m = Block(torch)
    scratch = lily.SamplerScratch(m.vocab, max_rows=rows, max_history=1024)
    lists, masks = _lists(torch, m, rows, 6)
    params, steps = _params(lily, rows), list(range(rows))
    wants = []
    for seed in (1, 2, 3):
        s = State(torch, m, tokens, rows)
        s.fill(torch, seed)
        _step(lily, scratch, m, s, params, lists, masks, steps)
        wants.append(s)
    s = State(torch, m, tokens, rows)
    s.fill(torch, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _step(lily, scratch, m, s, params, lists, masks, steps)
    for seed, want in zip((1, 2, 3), wants):
        s.fill(torch, seed)
        graph.replay()
        for name in ("sum", "y8_scales", "act", "out", "last", "logits", "adjusted", "ids", "status"):
            assert torch.equal(getattr(s, name), getattr(want, name)), name
    assert scratch.status() == lily.OK


def test_shards_draw_with_lists_and_masks(cuda, lily):
    """The whole row's draw with its lists and masks, and the shards' draw from adjusted shards: the same tokens;
    the sharded step does the same for a world of one."""
    import lily_b200.shard as sh

    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(31)
    vocab, hidden, rows, shards = 8000, 512, 6, 4
    w = torch.randint(-127, 128, (vocab, hidden), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    sc = (0.002 + 0.01 * torch.rand((vocab, hidden // 64), generator=g, device="cuda")).bfloat16()
    h = torch.randn((rows, hidden), generator=g, device="cuda").bfloat16()
    params, steps = _params(lily, rows), list(range(rows))
    m = Block(torch)
    m.vocab = vocab
    lists, masks = _lists(torch, m, rows, 7)
    whole = lily.SamplerScratch(vocab, max_rows=rows, max_history=1024, lmhead=True)
    logits, adjusted = torch.empty((rows, vocab), device="cuda"), torch.empty((rows, vocab), device="cuda")
    want, got = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    draw = [lily.draft_params(p) for p in params]
    whole.lmhead_logits(w, sc, h, logits)
    whole.adjust_logits(logits, params, adjusted, **lists, **masks)
    whole.sample_batch(adjusted, draw, want, steps=steps)

    per = vocab // shards
    part = lily.SamplerScratch(per, max_rows=rows, max_history=1024)
    records = torch.empty((shards, rows, sh.RECORD_BYTES), dtype=torch.uint8, device="cuda")
    for k in range(shards):
        mine = logits[:, k * per:(k + 1) * per].contiguous()
        part.adjust_logits(mine, params, first_id=k * per, **lists, **masks)
        assert torch.equal(mine, adjusted[:, k * per:(k + 1) * per])
        part.shard_candidates(mine, draw, records[k], first_id=k * per)
    part.merge_draw(records, draw, got, steps=steps)
    assert torch.equal(got, want)

    # The step of one rank, on a stream of its own too, with a buffer of the caller's.
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for kw in ({}, {"stream": side}, {"logits": torch.empty_like(logits)}):
        got.zero_()
        side.wait_stream(torch.cuda.current_stream())
        sh.sharded_lmhead_draw(whole, w, sc, h, params, got, 0, steps=steps, adjust={**lists, **masks}, **kw)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert whole.status() == part.status() == lily.OK
