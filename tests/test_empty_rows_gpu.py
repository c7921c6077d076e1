"""Greedy rows that a mask or bans have left with nothing: their draw says so (LILY_ROW_NONFINITE, no id), as a
sampled row's does and as a greedy row's does with the bans in its own call; by shards too, with the sums of
exponentials beside. The exact argmax (lily_argmax_batch) stays what it is.

out_lse: a term's argument is rounded three times at magnitudes below 64 (3 * 64 * 2^-24 * ln 2 < 2^-16.9), its
exponential and the sums' trees are below 2^-19, logf and the last sum below 2^-19 of |lse| < 64: 2^-14 in all."""
import numpy as np
import pytest

from gpu_util import np_u32

pytestmark = pytest.mark.gpu

NONE = 0xFFFFFFFF
GREEDY = [dict(temperature=0.0), dict(temperature=0.8, top_k=1), dict(temperature=0.0, top_k=40)]


def _words(torch, bits):
    """int32 words of [rows, ids] truth values."""
    rows, n = bits.shape
    full = np.zeros((rows, (n + 31) // 32 * 32), dtype=np.uint64)
    full[:, :n] = bits
    words = (full.reshape(rows, -1, 32) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32)
    return torch.from_numpy(words.view(np.int32)).cuda()


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 777), (3, 4096), (1, 151_936), (6, 20_000), (40, 5_000), (200, 9_000),
                                        (160, 70_000)])
@pytest.mark.parametrize("bf16", [False, True])
def test_greedy_rows_left_with_nothing(cuda, lily, rows, vocab, bf16):
    torch = cuda
    rng = np.random.default_rng([rows, vocab, bf16])
    scratch = lily.SamplerScratch(vocab, max_rows=rows)
    logits = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32)).cuda()
    logits = logits.bfloat16() if bf16 else logits
    bits = rng.random((rows, vocab)) < 0.5
    empty = np.arange(rows) % 3 == 0
    bits[empty] = False
    bits[~empty, rng.integers(0, vocab, int((~empty).sum()))] = True
    scratch.adjust_logits(logits, mask=_words(torch, bits))
    want = torch.argmax(logits.float(), 1).cpu().numpy()
    for p in GREEDY:
        out, status, kept_n = (torch.full((rows,), 77, dtype=torch.int32, device="cuda") for _ in range(3))
        kept = dict(kept_n=kept_n, kept_ids=torch.zeros((rows, lily.K_CAP), dtype=torch.int32, device="cuda"),
                    kept_probs=torch.zeros((rows, lily.K_CAP), device="cuda"))
        for kw in ({}, kept):
            scratch.sample_batch(logits, [lily.SamplingParams(**p)] * rows, out, uniforms=torch.zeros(rows, device="cuda"),
                                 out_status=status, **kw)
            got, said = np_u32(out), np_u32(status)
            assert (got[empty] == NONE).all() and (said[empty] == lily.ROW_NONFINITE).all(), p
            assert (said[~empty] == 0).all() and bits[~empty, got[~empty]].all()
            values = logits.float().cpu().numpy()
            assert (values[~empty, got[~empty]] == values[~empty, want[~empty]]).all()
            assert scratch.status() == lily.ERR_DEVICE_ROW and scratch.status() == lily.OK
        assert (np_u32(kept_n) == np.where(empty, 0, 1)).all()
    # The argmax of a row is an id, whatever its logits are.
    out = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    scratch.argmax_batch(logits, out)
    assert (np_u32(out)[empty] < vocab).all() and scratch.status() == lily.OK


@pytest.mark.parametrize("vocab", [300, 4096, 40_000])
def test_greedy_rows_of_nan(cuda, lily, vocab):
    """A NaN never wins. Rows of nothing else have an argmax all the same, but no id whose logit is -inf is drawn."""
    torch = cuda
    scratch = lily.SamplerScratch(vocab, max_rows=4)
    logits = torch.full((4, vocab), float("-inf"), device="cuda")
    logits[0] = float("nan")
    logits[1, vocab // 2] = float("nan")
    logits[2, vocab // 3] = -5.0
    logits[2, vocab // 2] = float("nan")
    logits[3, ::2] = float("nan")
    out, status = (torch.full((4,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    scratch.sample_batch(logits, [lily.SamplingParams()] * 4, out, uniforms=torch.zeros(4, device="cuda"), out_status=status)
    got, said = np_u32(out), np_u32(status)
    assert got[0] == 0 and said[0] == 0 and got[2] == vocab // 3 and said[2] == 0
    for r in (1, 3):
        assert (got[r] == NONE and said[r] == lily.ROW_NONFINITE) or (said[r] == 0 and bool(torch.isnan(logits[r, int(got[r])])))


def test_a_speculative_step_with_an_empty_row(cuda, lily):
    torch = cuda
    vocab = 5000
    scratch = lily.SamplerScratch(vocab, max_rows=4)
    g = torch.Generator(device="cuda").manual_seed(3)
    logits = torch.randn((4, vocab), generator=g, device="cuda")
    best = torch.argmax(logits, 1).int()
    mask = torch.full((2, (vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
    mask[0] = 0
    for empty in range(4):
        mine = logits.clone()
        scratch.adjust_logits(mine, mask=mask, mask_rows=(torch.arange(4, device="cuda") != empty).int())
        out, accepted = torch.full((4,), 77, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        scratch.spec_verify(mine, lily.SamplingParams(), best[:3].contiguous(), out, accepted, step0=0, mode=lily.SPEC_GREEDY_MATCH)
        assert scratch.status() == lily.ERR_DEVICE_ROW
        assert int(accepted) == min(empty, 3)
        got = np_u32(out)
        assert got[empty] == NONE and (got[:empty] == np_u32(best)[:empty]).all()


@pytest.mark.parametrize("shards", [1, 4])
@pytest.mark.parametrize("rows", [1, 9, 64])
def test_shards_of_tight_masks(cuda, lily, shards, rows):
    """Masks that leave 1 to 20 ids, all of one shard's, one that leaves nothing, one that leaves all: drawn from
    the shards' records as from the whole row, with the logarithm of the sum."""
    import lily_b200.shard as sh

    torch = cuda
    vocab = 8000
    per = vocab // shards
    rng = np.random.default_rng([shards, rows])
    logits = torch.from_numpy((3 * rng.standard_normal((rows, vocab))).astype(np.float32)).cuda()
    bits = np.zeros((rows, vocab), dtype=bool)
    for r in range(rows):
        if r % 9 == 8:
            bits[r] = True
        elif r % 9 != 0 or rows == 1:
            at = int(rng.integers(0, shards)) * per
            bits[r, at + rng.choice(per, int(rng.integers(1, 21)), replace=False)] = True
    mask = _words(torch, bits)
    whole, part = lily.SamplerScratch(vocab, max_rows=rows), lily.SamplerScratch(per, max_rows=rows)
    scratch_rows = torch.empty_like(logits)
    whole.adjust_logits(logits, out=scratch_rows, mask=mask)
    empty = ~bits.any(1)
    draws = [dict(temperature=0.8, top_k=40, top_p=0.95), dict(temperature=1.3, top_k=64), dict(temperature=1.0, top_k=2), *GREEDY]
    for p in draws:
        params = [lily.SamplingParams(seed=r, **p) for r in range(rows)]
        u = torch.from_numpy(rng.random(rows).astype(np.float32)).cuda()
        want, got, want_status, status = (torch.full((rows,), 77, dtype=torch.int32, device="cuda") for _ in range(4))
        whole.sample_batch(scratch_rows, params, want, uniforms=u, out_status=want_status)
        whole.status()
        for want_sums in (False, True):
            records = torch.empty((shards, rows, sh.RECORD_BYTES), dtype=torch.uint8, device="cuda")
            lse = torch.full((rows,), 123.0, device="cuda")
            for k in range(shards):
                mine = logits[:, k * per:(k + 1) * per].contiguous()
                part.adjust_logits(mine, first_id=k * per, mask=mask)
                part.shard_candidates(mine, params, records[k], first_id=k * per, want_sums=want_sums)
            assert part.status() == lily.OK
            part.merge_draw(records, params, got, uniforms=u, out_status=status, out_lse=lse if want_sums else None)
            assert part.status() == (lily.ERR_DEVICE_ROW if empty.any() else lily.OK)
            assert torch.equal(got, want), (p, want_sums)
            assert torch.equal(status, want_status)
            assert (np_u32(got)[empty] == NONE).all() and (np_u32(status)[empty] == lily.ROW_NONFINITE).all()
            if want_sums:
                greedy = p["temperature"] == 0.0 or p.get("top_k") == 1
                exact = torch.logsumexp(scratch_rows.double() / (1.0 if greedy else p["temperature"]), 1)
                assert (lse.double() - exact).abs().nan_to_num(0.0)[~torch.from_numpy(empty).cuda()].max() <= 2.0 ** -14


@pytest.mark.parametrize("shards", [1, 2, 7])
def test_the_sum_of_nothing(cuda, lily, shards):
    """log 0 is -inf, from one shard's records and from several."""
    import lily_b200.shard as sh

    torch = cuda
    part = lily.SamplerScratch(1000, max_rows=3)
    for p in (dict(temperature=0.7, top_k=20), dict(temperature=0.0)):
        params = [lily.SamplingParams(**p)] * 3
        records = torch.empty((shards, 3, sh.RECORD_BYTES), dtype=torch.uint8, device="cuda")
        for k in range(shards):
            logits = torch.full((3, 1000), float("-inf"), device="cuda")
            logits[1, 17] = 2.0 if k == shards - 1 else float("-inf")
            part.shard_candidates(logits, params, records[k], first_id=1000 * k, want_sums=True)
        out, status = (torch.full((3,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
        lse = torch.full((3,), 123.0, device="cuda")
        part.merge_draw(records, params, out, uniforms=torch.zeros(3, device="cuda"), out_status=status, out_lse=lse)
        assert part.status() == lily.ERR_DEVICE_ROW
        assert status.tolist() == [lily.ROW_NONFINITE, 0, lily.ROW_NONFINITE]
        assert np_u32(out).tolist() == [NONE, 1000 * (shards - 1) + 17, NONE]
        assert torch.isneginf(lse[[0, 2]]).all(), lse
        assert abs(float(lse[1]) - 2.0 / (p["temperature"] or 1.0)) <= 2.0 ** -14
