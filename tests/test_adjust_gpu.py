"""lily_adjust_logits on the GPU against the formula in 64 bits, bit for bit against the same steps in
binary32 on the CPU, and against the draws that have penalties, biases and bans built in.

In 64 bits: an entry of a list, the penalty's product or quotient, presence + frequency * count (two) and
the subtraction each round once, 2^-24 of a value no larger than the sum of the magnitudes that went
in: with n bias entries (n + 4) * 2^-24 of it. bf16 adds half a step, 2^-8 of the result."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GUARD = 3.25


def _i32(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.uint32).view(np.int32)).cuda()


class Case:
    """A call's inputs on the host; lists may name an id twice, or ids outside the vocabulary."""

    def __init__(self, rng, rows, vocab, bf16, history=0, lists=0, masks=0, frequency=True, total=None, first=0):
        self.rows, self.vocab, self.bf16, self.first = rows, vocab, bf16, first
        total = total or vocab + first
        x = (rng.standard_normal((rows, vocab)) * 4).astype(np.float32)
        if bf16:
            x = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        self.logits = x
        self.params = None
        if history:
            # Skewed, so that ids come many times.
            self.history = (total * rng.random((rows, history)) ** 6).astype(np.uint32)
            self.history[:, ::17] = total + 5  # no such id
            self.history_len = rng.integers(0, history + 1, rows)
            self.history_len[0] = history
            self.params = [dict(temperature=0.7, top_k=20, top_p=0.95, repetition_penalty=[1.0, 1.3, 0.8][r % 3],
                                presence_penalty=[0.5, 0.0, -0.25][r % 3],
                                frequency_penalty=[0.1, 0.0, 0.3][r % 3] if frequency else 0.0, seed=r) for r in range(rows)]
        else:
            self.history = None
        self.bias = None
        if lists:
            self.bias = rng.integers(0, total + 3, (rows, lists))
            self.bias[:, 1::3] = self.bias[:, ::3][:, :self.bias[:, 1::3].shape[1]]  # the same id twice
            self.bias_vals = (rng.standard_normal((rows, lists)) * 3).astype(np.float32)
            self.bias_len = rng.integers(0, lists + 1, rows)
            self.ban = rng.integers(0, total + 3, (rows, lists))
            self.ban_len = rng.integers(0, lists + 1, rows)
            if rows > 1:
                self.ban[1, 0] = self.bias[1, 0]  # biased and banned
                self.ban_len[1] = self.bias_len[1] = lists
        self.mask = None
        if masks:
            words = (total + 31) // 32
            density = rng.choice([0.01, 0.5, 0.97], masks)[:, None, None]
            bits = rng.random((masks, words, 32)) < density
            if masks > 1:
                bits[1] = False  # leaves nothing
            self.bits = bits.reshape(masks, -1)
            self.mask = (bits.astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32)
            self.mask_rows = rng.integers(-1, masks, rows).astype(np.int32)
            if masks > 1 and rows > 2:
                self.mask_rows[2] = 1

    def args(self, torch, lily):
        kw = {"first_id": self.first}
        if self.history is not None:
            kw.update(history_ids=_i32(torch, self.history), history_len=_i32(torch, self.history_len))
        if self.bias is not None:
            kw.update(bias_ids=_i32(torch, self.bias), bias_vals=torch.from_numpy(self.bias_vals).cuda(),
                      bias_len=_i32(torch, self.bias_len), ban_ids=_i32(torch, self.ban), ban_len=_i32(torch, self.ban_len))
        if self.mask is not None:
            kw.update(mask=_i32(torch, self.mask), mask_rows=torch.from_numpy(self.mask_rows).cuda())
        return kw, None if self.params is None else [lily.SamplingParams(**p) for p in self.params]

    def expected(self, real):
        """The formula row by row in `real` (np.float32: with the kernel's order of operations), and the
        sum of magnitudes that went into each value."""
        out, size = self.logits.astype(real), np.abs(self.logits.astype(np.float64))
        for r in range(self.rows):
            l = out[r]
            if self.bias is not None:
                for i, v in zip(self.bias[r, :self.bias_len[r]], self.bias_vals[r]):
                    if self.first <= i < self.first + self.vocab:
                        l[i - self.first] = l[i - self.first] + real(v)
                        size[r, i - self.first] += abs(float(v))
            if self.history is not None:
                p = self.params[r]
                rep, pres, freq = (real(np.float32(p[k])) for k in ("repetition_penalty", "presence_penalty",
                                                                    "frequency_penalty"))
                ids = self.history[r, :self.history_len[r]].astype(np.int64) - self.first
                ids, count = np.unique(ids[(ids >= 0) & (ids < self.vocab)], return_counts=True)
                if rep != 1 or pres != 0 or freq != 0:
                    v = l[ids]
                    v = np.where(v > 0, v / rep, v * rep)
                    s = pres + freq * count.astype(real)
                    l[ids] = v - s
                    size[r, ids] = size[r, ids] * 1.3 + np.abs(s)
            if self.bias is not None:
                for i in self.ban[r, :self.ban_len[r]]:
                    if self.first <= i < self.first + self.vocab:
                        l[i - self.first] = -np.inf
            if self.mask is not None and self.mask_rows[r] >= 0:
                l[~self.bits[self.mask_rows[r], self.first:self.first + self.vocab]] = -np.inf
        return out, size


def _run(torch, lily, scratch, case, out_f32, in_place, pitch=0, offset=0):
    """The adjusted logits as float32 on the host; rows `pitch` apart, `offset` elements into their buffers."""
    t_in = torch.bfloat16 if case.bf16 else torch.float32
    t_out = torch.float32 if out_f32 else t_in
    ld = case.vocab + pitch
    size = offset + case.rows * ld + 8

    def place(t):
        buf = torch.full((size,), GUARD, dtype=t, device="cuda")
        return buf, buf[offset:offset + case.rows * ld].view(case.rows, ld)[:, :case.vocab]

    buf, logits = place(t_in)
    logits.copy_(torch.from_numpy(case.logits))
    out_buf, out = (buf, logits) if in_place else place(t_out)
    kw, params = case.args(torch, lily)
    status = torch.full((case.rows,), 77, dtype=torch.int32, device="cuda")
    scratch.adjust_logits(logits, params, None if in_place else out, out_status=status, **kw)
    assert (status == 0).all()
    outside = torch.ones(size, dtype=torch.bool, device="cuda")
    outside[offset:offset + case.rows * ld].view(case.rows, ld)[:, :case.vocab] = False
    assert (out_buf[outside] == GUARD).all(), "written outside the rows"
    return out.float().cpu().numpy()


def _check(case, got, rounded):
    want, size = case.expected(np.float64)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    fine = np.isfinite(want)
    n = 0 if case.bias is None else case.bias.shape[1]
    tol = (n + 4) * 2.0 ** -24 * size + (2.0 ** -8 * np.abs(np.where(fine, want, 0.0)) if rounded else 0.0) * 1.01
    assert (np.abs(got.astype(np.float64) - np.where(fine, want, 0.0))[fine] <= tol[fine]).all()
    if not rounded:
        same, _ = case.expected(np.float32)
        assert np.array_equal(got.view(np.uint32), same.view(np.uint32))


SHAPES = [(1, 1), (1, 33), (2, 255), (3, 257), (1, 4096), (5, 4099), (4, 50257), (3, 32768), (2, 100_000), (40, 5000), (300, 777)]


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("bf16", [False, True])
def test_everything_on(cuda, lily, rows, vocab, bf16):
    rng = np.random.default_rng([rows, vocab, bf16])
    scratch = lily.SamplerScratch(vocab, max_rows=rows, max_history=4096, max_list=64)
    for history, lists, masks in ((1000, 20, 3), (0, 0, 4), (777, 0, 0), (0, 5, 0), (4096, 64, 2)):
        case = Case(rng, rows, vocab, bf16, history, lists, masks)
        for out_f32, in_place in ((True, False), (False, False), (False, True)):
            _check(case, _run(cuda, lily, scratch, case, out_f32, in_place), bf16 and not out_f32)
    assert scratch.status() == 0


@pytest.mark.parametrize("pitch,offset", [(0, 0), (8, 0), (8, 8), (1, 0), (5, 3), (16, 1), (0, 4)])
def test_rows_of_any_pitch_and_alignment(cuda, lily, pitch, offset):
    rng = np.random.default_rng([pitch, offset])
    vocab = 9000
    scratch = lily.SamplerScratch(vocab, max_rows=4, max_history=500, max_list=16)
    for bf16 in (False, True):
        case = Case(rng, 4, vocab, bf16, 500, 16, 2, frequency=False)
        for out_f32, in_place in ((True, False), (False, False), (False, True)):
            _check(case, _run(cuda, lily, scratch, case, out_f32, in_place, pitch, offset), bf16 and not out_f32)


@pytest.mark.parametrize("shards,vocab", [(2, 8192), (3, 3 * 1111), (8, 8 * 1000), (7, 7 * 4097)])
def test_shards_put_together_are_the_whole_row(cuda, lily, shards, vocab):
    rng = np.random.default_rng([shards, vocab])
    whole = Case(rng, 5, vocab, False, 800, 24, 3)
    want, _ = whole.expected(np.float32)
    here = vocab // shards
    scratch = lily.SamplerScratch(here, max_rows=5, max_history=800, max_list=24)
    kw, params = whole.args(cuda, lily)
    logits = cuda.from_numpy(whole.logits).cuda()
    for s in range(shards):
        kw["first_id"] = s * here
        part = logits[:, s * here:(s + 1) * here]
        scratch.adjust_logits(part, params, **kw)  # (in place, rows a vocabulary apart)
    assert np.array_equal(logits.cpu().numpy().view(np.uint32), want.view(np.uint32))
    assert scratch.status() == 0


@pytest.mark.parametrize("bf16", [False, True])
def test_the_draw_behind_it_is_the_draw_with_everything_in_one(cuda, lily, bf16):
    torch = cuda
    rng = np.random.default_rng([9, bf16])
    rows, vocab = 12, 20_000
    case = Case(rng, rows, vocab, bf16, 1500, 32, 0)
    scratch = lily.SamplerScratch(vocab, max_rows=rows, max_history=1500, max_list=32)
    kw, params = case.args(torch, lily)
    kw.pop("first_id")
    t = torch.from_numpy(case.logits).cuda()
    logits = t.bfloat16() if bf16 else t
    u = torch.from_numpy(rng.random(rows).astype(np.float32)).cuda()
    one, two = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    scratch.sample_batch(logits, params, one, uniforms=u, **kw)
    adjusted = torch.empty((rows, vocab), device="cuda")
    scratch.adjust_logits(logits, params, adjusted, **kw)
    scratch.sample_batch(adjusted, [lily.draft_params(p) for p in params], two, uniforms=u)
    assert torch.equal(one, two)
    # A mask of one id leaves that id to every draw.
    only = rng.integers(0, vocab, rows)
    bits = np.zeros((rows, (vocab + 31) // 32 * 32), dtype=np.uint64)
    bits[np.arange(rows), only] = 1
    mask = (bits.reshape(rows, -1, 32) << np.arange(32, dtype=np.uint64)).sum(2)
    scratch.adjust_logits(adjusted, mask=_i32(torch, mask))
    keep = torch.isfinite(adjusted).any(1).cpu().numpy()  # (unless a list has banned it)
    scratch.sample_batch(adjusted, [lily.draft_params(p) for p in params], two, uniforms=u)
    assert np.array_equal(two.cpu().numpy()[keep], only[keep]) and keep.sum() >= rows - 2


def test_a_mask_that_leaves_nothing_and_values_under_masks(cuda, lily):
    torch = cuda
    vocab = 3000
    scratch = lily.SamplerScratch(vocab, max_rows=3)
    logits = torch.randn((3, vocab), device="cuda")
    logits[0, :] = float("nan")
    logits[1, 10:20] = float("inf")
    logits[1, 20:30] = float("nan")
    logits[2, :] = torch.finfo(torch.float32).min
    mask = torch.full((2, (vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
    mask[0] = 0
    mask[1, 0] = -(1 << 30)  # ids 30 and 31 of the first 32
    scratch.adjust_logits(logits, mask=mask, mask_rows=torch.tensor([0, 1, -1], dtype=torch.int32, device="cuda"))
    assert torch.isneginf(logits[0]).all()
    assert torch.isneginf(logits[1, :30]).all() and torch.isfinite(logits[1, 30:]).all()
    assert (logits[2] == torch.finfo(torch.float32).min).all()
    out, status = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2))
    p = lily.SamplingParams(temperature=1.0, top_k=20, top_p=0.9)
    scratch.sample_batch(logits, [p] * 3, out, uniforms=torch.full((3,), 0.5, device="cuda"), out_status=status)
    assert status.tolist() == [lily.ROW_NONFINITE, 0, 0]
    assert scratch.status() == lily.ERR_DEVICE_ROW


def test_counts_beyond_sixteen_bits(cuda, lily):
    torch = cuda
    vocab, n = 2000, 70_000
    scratch = lily.SamplerScratch(vocab, max_rows=2, max_history=n)
    logits = torch.zeros((2, vocab), device="cuda")
    history = torch.full((2, n), 1234, dtype=torch.int32, device="cuda")
    history[1, :10] = 5
    params = [lily.SamplingParams(frequency_penalty=0.5)] * 2
    scratch.adjust_logits(logits, params, history_ids=history,
                          history_len=torch.tensor([n, 65_546], dtype=torch.int32, device="cuda"))
    want = torch.zeros((2, vocab), device="cuda")
    want[0, 1234], want[1, 1234], want[1, 5] = -0.5 * n, -0.5 * 65_536, -5.0
    assert torch.equal(logits, want)


@pytest.mark.parametrize("rows,vocab,history", [(300, 40_000, 16_000), (100, 30_001, 9_000), (1, 9_000, 9_000), (150, 21_000, 30_000)])
def test_more_ids_than_a_block_counts_at_a_time(cuda, lily, rows, vocab, history):
    """Histories of all different ids, and of a row's whole vocabulary."""
    rng = np.random.default_rng([rows, vocab])
    case = Case(rng, rows, vocab, True, history, 12, 2)
    for r in range(rows):  # (uniform: nearly all of them different)
        case.history[r] = rng.integers(0, vocab, history)
    case.history[0, :min(vocab, history)] = rng.permutation(vocab)[:history]
    case.bias[:, 0] = case.history[:, history // 2]
    case.bias_len[:] = 12
    scratch = lily.SamplerScratch(vocab, max_rows=rows, max_history=history, max_list=12)
    for out_f32, in_place in ((True, False), (False, True)):
        _check(case, _run(cuda, lily, scratch, case, out_f32, in_place), not out_f32)


def test_histogram_slots_with_masks_and_biases(cuda, lily):
    torch = cuda
    rng = np.random.default_rng(14)
    rows, vocab = 4, 30_007
    case = Case(rng, rows, vocab, False, 0, 20, 2)
    counts = (rng.random((rows, vocab)) < 0.3) * rng.integers(1, 70_000, (rows, vocab))
    case.bias[:, 1] = np.argmax(counts > 0, axis=1)
    scratch = lily.SamplerScratch(vocab, max_rows=rows, max_list=20, counts_table=True)
    for s in range(rows):
        scratch.write_counts(counts[s].astype(np.uint32), slot=s)
    kw, _ = case.args(torch, lily)
    params = [lily.SamplingParams(repetition_penalty=1.25, frequency_penalty=0.5, presence_penalty=0.125)] * rows
    x = case.logits.copy()
    for r in range(rows):
        for i, v in zip(case.bias[r, :case.bias_len[r]], case.bias_vals[r]):
            if i < vocab:
                x[r, i] = x[r, i] + v
    c = counts.astype(np.float32)
    want = np.where(counts > 0, np.where(x > 0, x / np.float32(1.25), x * np.float32(1.25)) - (np.float32(0.125) + np.float32(0.5) * c), x)
    for r in range(rows):
        want[r, [i for i in case.ban[r, :case.ban_len[r]] if i < vocab]] = -np.inf
        if case.mask_rows[r] >= 0:
            want[r, ~case.bits[case.mask_rows[r], :vocab]] = -np.inf
    for in_place in (False, True):
        logits = torch.from_numpy(case.logits).cuda()
        out = logits if in_place else torch.empty_like(logits)
        scratch.adjust_logits(logits, params, None if in_place else out, count_slots=list(range(rows)), **kw)
        assert np.array_equal(out.cpu().numpy().view(np.uint32), want.astype(np.float32).view(np.uint32))
    assert scratch.status() == 0


def test_histogram_slots(cuda, lily):
    torch = cuda
    rng = np.random.default_rng(4)
    for vocab in (1000, 40_003):
        scratch = lily.SamplerScratch(vocab, max_rows=3, counts_table=True)
        counts = (rng.random((3, vocab)) < 0.1) * rng.integers(1, 9, (3, vocab))
        for s in range(3):
            scratch.write_counts(counts[s].astype(np.uint32), slot=s)
        x = rng.standard_normal((2, vocab)).astype(np.float32)
        params = [lily.SamplingParams(repetition_penalty=1.25, frequency_penalty=0.5, presence_penalty=0.125)] * 2
        out = torch.empty((2, vocab), device="cuda")
        scratch.adjust_logits(torch.from_numpy(x).cuda(), params, out, count_slots=[2, 0])
        c = counts[[2, 0]]
        v = np.where(x > 0, x / np.float32(1.25), x * np.float32(1.25)) - (np.float32(0.125) + np.float32(0.5) * c.astype(np.float32))
        want = np.where(c > 0, v, x).astype(np.float32)
        assert np.array_equal(out.cpu().numpy().view(np.uint32), want.view(np.uint32))
        for s in range(3):
            assert np.array_equal(scratch.read_counts(slot=s), counts[s])


def test_parameters_on_the_device(cuda, lily):
    torch = cuda
    rng = np.random.default_rng(6)
    rows, vocab = 5, 6000
    case = Case(rng, rows, vocab, False, 300, 8, 2)
    scratch = lily.SamplerScratch(vocab, max_rows=rows, max_history=300, max_list=8)
    kw, params = case.args(torch, lily)
    params[3].repetition_penalty = -1.0  # not valid: its row is left as it is
    raw = torch.from_numpy(np.frombuffer(b"".join(bytes(p) for p in params), dtype=np.uint8).copy()).cuda()
    out = torch.full((rows, vocab), GUARD, device="cuda")
    status = torch.zeros(rows, dtype=torch.int32, device="cuda")
    scratch.adjust_logits(torch.from_numpy(case.logits).cuda(), raw, out, params_on_device=True, out_status=status, **kw)
    want, _ = case.expected(np.float32)
    want[3] = GUARD
    assert status.tolist() == [0, 0, 0, lily.ROW_PARAMS, 0]
    assert np.array_equal(out.cpu().numpy().view(np.uint32), want.view(np.uint32))
    assert scratch.status() == lily.ERR_DEVICE_ROW


def test_rows_whose_lists_are_too_long_are_left_alone(cuda, lily):
    torch = cuda
    vocab = 2048
    scratch = lily.SamplerScratch(vocab, max_rows=4, max_history=64, max_list=8)
    logits = torch.ones((4, vocab), device="cuda")
    history = torch.zeros((4, 64), dtype=torch.int32, device="cuda")
    ban = torch.ones((4, 8), dtype=torch.int32, device="cuda")
    mask = torch.zeros((1, vocab // 32), dtype=torch.int32, device="cuda")
    status = torch.zeros(4, dtype=torch.int32, device="cuda")
    as_i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    scratch.adjust_logits(logits, [lily.SamplingParams(presence_penalty=1.0)] * 4, history_ids=history,
                          history_len=as_i32(64, 65, -1, 3), ban_ids=ban, ban_len=as_i32(8, 0, 0, 9), mask=mask,
                          mask_rows=as_i32(-1, -1, -1, -1), out_status=status)
    assert status.tolist() == [0, lily.ROW_LIST, lily.ROW_LIST, lily.ROW_LIST]
    assert (logits[1:] == 1).all() and logits[0, 0] == 0 and torch.isneginf(logits[0, 1])
    assert scratch.status() == lily.ERR_DEVICE_ROW
    scratch.adjust_logits(logits, mask=mask, mask_rows=as_i32(-1, 1, 0, -5), out_status=status)
    assert status.tolist() == [0, lily.ROW_LIST, 0, 0]
    assert torch.isneginf(logits[2]).all() and (logits[1] == 1).all() and (logits[3] == 1).all()


def test_captured_and_side_by_side(cuda, lily):
    """Two captured calls of one handle replayed on two streams: nothing is shared between them."""
    torch = cuda
    rng = np.random.default_rng(12)
    rows, vocab = 6, 30_000
    scratch = lily.SamplerScratch(vocab, max_rows=rows, max_history=2000, max_list=16)
    runs = []
    for _ in range(2):
        case = Case(rng, rows, vocab, False, 2000, 16, 3)
        kw, params = case.args(torch, lily)
        logits, out = torch.from_numpy(case.logits).cuda(), torch.empty((rows, vocab), device="cuda")
        scratch.adjust_logits(logits, params, out, **kw)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scratch.adjust_logits(logits, params, out, **kw)
        runs.append((case, graph, out, torch.cuda.Stream(), (kw, logits)))
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(10):
        for _, graph, _, stream, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for case, _, out, _, _ in runs:
        assert np.array_equal(out.cpu().numpy().view(np.uint32), case.expected(np.float32)[0].view(np.uint32))


def test_refusals(cuda, lily):
    torch = cuda
    vocab = 1000
    scratch = lily.SamplerScratch(vocab, max_rows=2)
    logits = torch.zeros((2, vocab), device="cuda")
    ids = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    mask = torch.zeros((2, 32), dtype=torch.int32, device="cuda")
    good = [lily.SamplingParams()] * 2
    for kw in (dict(logits=logits.cpu()), dict(logits=logits[:, :999]), dict(logits=logits.half()),
               dict(out=torch.zeros((2, vocab), dtype=torch.bfloat16, device="cuda")), dict(out=logits[:1]),
               dict(params=good[:1]), dict(history_ids=ids), dict(bias_ids=ids, bias_len=n), dict(ban_len=n),
               dict(mask=mask[:, :31]), dict(mask=mask[:1]), dict(mask=mask, first_id=100), dict(mask_rows=n),
               dict(mask=mask.float()), dict(first_id=1 << 32), dict(first_id=-1), dict(first_id=0xFFFFFFFF),
               dict(count_slots=[0, 1]), dict(history_ids=ids, history_len=n[:1]), dict(history_ids=ids[:1], history_len=n),
               dict(logits=torch.zeros((3, vocab), device="cuda"))):
        call = {"logits": logits, **kw}
        with pytest.raises(lily.LilyError) as e:
            scratch.adjust_logits(call.pop("logits"), call.pop("params", None), call.pop("out", None), **call)
        assert e.value.code in (lily.ERR_ARG, lily.ERR_CAPACITY), kw
    bad = lily.SamplingParams()
    bad.repetition_penalty = 0.0
    with pytest.raises(lily.LilyError) as e:
        scratch.adjust_logits(logits, [good[0], bad])
    assert e.value.code == lily.ERR_PARAMS
    with pytest.raises(TypeError):
        scratch.adjust_logits(logits, bias=1)
    # An empty list is no list.
    empty = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    scratch.adjust_logits(logits, good, history_ids=empty, history_len=n)
    assert (logits == 0).all() and scratch.status() == lily.OK


def test_misaligned_lists_are_refused(cuda, lily):
    """By the host, before anything is enqueued."""
    import ctypes as C

    torch = cuda
    scratch = lily.SamplerScratch(1000, max_rows=2)
    logits, words = torch.zeros((2, 1000), device="cuda"), torch.zeros(4096, dtype=torch.int32, device="cuda")
    device_params = torch.zeros(2 * C.sizeof(lily.SamplingParams) + 1, dtype=torch.uint8, device="cuda")
    with pytest.raises(lily.LilyError) as e:
        scratch.adjust_logits(logits, device_params[1:], params_on_device=True)
    assert e.value.code == lily.ERR_ARG
    fields = ("history_ids", "history_len", "bias_ids", "bias_vals", "bias_len", "ban_ids", "ban_len", "mask", "mask_rows",
              "out_status")
    for off in (None, *fields):
        a = lily.AdjustArgs()
        a.struct_size, a.rows = C.sizeof(lily.AdjustArgs), 2
        a.logits = a.out = logits.data_ptr()
        a.logits_ld = a.out_ld = 1000
        for name in fields:
            setattr(a, name, words.data_ptr() + (2 if name == off else 0))
        a.history_ld = a.bias_ld = a.ban_ld = 4
        a.mask_ld, a.masks = 32, 2
        st = lily.lib().lily_adjust_logits(scratch._h, torch.cuda.current_stream().cuda_stream, C.byref(a))
        assert st == (lily.OK if off is None else lily.ERR_ARG), off


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_beyond_32_bits(cuda, lily, bf16):
    """Rows of logits more than 2^32 bytes apart; the last one is adjusted as it is alone."""
    torch = cuda
    rng = np.random.default_rng(77)
    vocab, rows, pitch = 5001, 3, 2 ** 31 + 8
    case = Case(rng, rows, vocab, bf16, history=300, lists=8, masks=2)
    dtype = torch.bfloat16 if bf16 else torch.float32
    buffer = torch.empty((rows - 1) * pitch + vocab, dtype=dtype, device="cuda")
    far = buffer.as_strided((rows, vocab), (pitch, 1))
    near = torch.from_numpy(case.logits).cuda().to(dtype)
    far.copy_(near)
    scratch = lily.SamplerScratch(vocab, max_rows=rows, max_history=512)
    kw, params = case.args(torch, lily)
    scratch.adjust_logits(near, params, **kw)
    scratch.adjust_logits(far, params, **kw)
    assert torch.equal(far, near)
    assert scratch.status() == lily.OK
