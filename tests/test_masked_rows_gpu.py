"""Draws from rows of which little is left: fewer finite logits than the candidate set takes, as a
grammar's mask leaves them. The k-th largest logit is then -inf, whatever route the row takes."""
import numpy as np
import pytest

import oracle
from gpu_util import np_u32, t_f32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab", [(1, 20_000), (12, 20_000), (5, 151_936), (200, 9_000), (160, 70_000)])
@pytest.mark.parametrize("bf16", [False, True])
def test_rows_of_fewer_finite_logits_than_candidates(cuda, lily, rows, vocab, bf16):
    torch = cuda
    rng = np.random.default_rng([rows, vocab, bf16])
    scratch = lily.SamplerScratch(vocab, max_rows=rows)
    check = list(range(min(rows, 4))) + ([rows - 1] if rows > 4 else [])
    for finite in (1, 2, 19, 20, 21, 700):
        for level in (4.0, -4.0):
            x = np.full((rows, vocab), -np.inf, dtype=np.float32)
            for r in range(rows):
                ids = rng.choice(vocab, finite, replace=False)
                x[r, ids] = (level + rng.standard_normal(finite)).astype(np.float32)
            if bf16:
                x = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
            logits = t_f32(torch, x)
            logits = logits.bfloat16() if bf16 else logits
            u = rng.random(rows).astype(np.float32)
            out, status = (torch.full((rows,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
            for p in (dict(temperature=0.7, top_k=20, top_p=0.95), dict(temperature=1.3, top_k=64), dict(temperature=0.0),
                      dict(temperature=1.0, top_k=0, top_p=0.9)):
                scratch.sample_batch(logits, [lily.SamplingParams(**p)] * rows, out, uniforms=t_f32(torch, u), out_status=status)
                assert (status == 0).all(), (finite, level, p)
                got = np_u32(out)
                assert np.isfinite(x[np.arange(rows), got]).all()
                for r in check:
                    assert got[r] == oracle.sample(x[r], oracle.params(**p), float(u[r]), mode=1).token, (finite, level, p, r)
    assert scratch.status() == lily.OK
