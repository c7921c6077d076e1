"""Rows of which next to nothing is left tie by the thousands at -inf, more than the candidate buffer takes: the row
is streamed again, from what its lists had pushed. Many such rows, launch after launch, drawn whole and as a shard's
records (how a block's warps come to the pass differs from launch to launch)."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,dtype", [(592, 4608, "float32"), (600, 8700, "bfloat16"), (300, 20_000, "float32"), (271, 4964, "float32"),
                                              (271, 7696, "float32"), (300, 8100, "float32"), (300, 11_000, "float32")])
def test_rows_of_ties_again_and_again(cuda, lily, rows, vocab, dtype):
    import lily_b200.shard as sh

    torch = cuda
    scratch = lily.SamplerScratch(vocab, max_rows=rows, max_list=4)
    logits = torch.full((rows, vocab), float("-inf"), device="cuda", dtype=getattr(torch, dtype))
    logits[1::2, 77] = -3.0
    params = [lily.SamplingParams(temperature=0.9, top_k=20)] * rows
    records = torch.empty((rows, sh.RECORD_BYTES), dtype=torch.uint8, device="cuda")
    out, status = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    u = torch.rand(rows, device="cuda")
    banned = dict(ban_ids=torch.full((rows, 1), 78, dtype=torch.int32, device="cuda"),
                  ban_len=torch.ones(rows, dtype=torch.int32, device="cuda"))
    even = torch.arange(rows, device="cuda") % 2 == 0
    wrong = torch.zeros(3, dtype=torch.int64, device="cuda")
    for _ in range(2500):
        scratch.shard_candidates(logits, params, records, first_id=0)
        best = records[:, 512:516].contiguous().view(torch.float32)[:, 0]
        wrong[0] += (best[even] != float("-inf")).sum() + ((best[~even] + 3.0 / 0.9).abs() > 1e-6).sum()
        for i, kw in ((1, {}), (2, banned)):
            scratch.sample_batch(logits, params, out, uniforms=u, out_status=status, **kw)
            wrong[i] += (status[even] != lily.ROW_NONFINITE).sum() + (status[~even] != 0).sum() + (out[~even] != 77).sum()
    assert wrong.tolist() == [0, 0, 0]
