"""What a sharded step on a stream of its own allocates is that stream's memory: the allocator gives it to nobody else
while the step's work is still to run."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("adjusted", [False, True])
def test_buffers_belong_to_the_step_s_stream(cuda, lily, adjusted, monkeypatch):
    import lily_b200.shard as sh

    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(2)
    vocab, hidden, rows = 4000, 512, 3
    w = torch.randint(-127, 128, (vocab, hidden), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    sc = (0.002 + 0.01 * torch.rand((vocab, hidden // 64), generator=g, device="cuda")).bfloat16()
    h = torch.randn((rows, hidden), generator=g, device="cuda").bfloat16()
    scratch = lily.SamplerScratch(vocab, max_rows=rows, lmhead=True)
    params, want, got = [lily.SamplingParams(temperature=0.9, top_k=30)] * rows, *(torch.zeros(rows, dtype=torch.int32, device="cuda")
                                                                                    for _ in range(2))
    kw = dict(steps=[1, 2, 3], adjust={"mask": torch.full((rows, 125), 0x55555555, dtype=torch.int32, device="cuda")} if adjusted else None)
    sh.sharded_lmhead_draw(scratch, w, sc, h, params, want, 0, **kw)
    torch.cuda.synchronize()
    side, empty, made = torch.cuda.Stream(), torch.empty, []

    def watched(*a, **k):
        t = empty(*a, **k)
        if t.is_cuda:
            made.append(torch.cuda.current_stream())
        return t

    monkeypatch.setattr(torch, "empty", watched)
    sh.sharded_lmhead_draw(scratch, w, sc, h, params, got, 0, stream=side, **kw)
    monkeypatch.undo()
    torch.cuda.synchronize()
    assert made and all(s == side for s in made), made
    assert torch.equal(got, want) and scratch.status() == lily.OK
