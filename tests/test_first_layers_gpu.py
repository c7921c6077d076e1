"""The first norm, product and adjustment of a kind in a process, captured or not: as for the draws, what they run is on
the device when the handle is made. In processes of their own, whose first calls these are."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = '''
import sys
import torch
import lily_b200 as lily

VOCAB, ROWS = 9000, 40
g = torch.Generator(device="cuda").manual_seed(5)
rand = lambda *s, t=torch.float32: torch.randn(s, generator=g, device="cuda").to(t)
full = lambda shape, v: torch.full(shape, v, dtype=torch.int32, device="cuda")
F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn

def calls(s):
    """(name, call, its outputs)"""
    for tokens in (3, 700):
        for hidden in (200, 512, 1000, 1001, 4096, 8192, 20000):
            for x_type in (F32, BF16):
                x, w = rand(tokens, hidden, t=x_type), rand(hidden)
                for out_type in (F32, BF16, E4M3):
                    for pad in (0, 1):
                        out = torch.zeros((tokens, hidden + pad), dtype=out_type, device="cuda")[:, :hidden]
                        kw = {"out_scales": torch.empty(tokens, device="cuda")} if out_type == E4M3 else {}
                        yield (f"norm {tokens} {hidden} {x_type} {out_type} {pad}", lambda st, x=x, w=w, o=out, kw=kw:
                               s.add_rms_norm(x, w, o, stream=st, **kw), out)
    for kind in (BF16, E4M3):
        for tokens in (3, 20, 40, 300):
            for outputs in (300, 20000):
                a, w = (rand(n, 512, t=kind) for n in (tokens, outputs))
                kw = {} if kind == BF16 else dict(a_scales=rand(tokens), weight_scales=rand(outputs))
                out = torch.zeros((tokens, outputs), device="cuda")
                yield (f"product {kind} {tokens} {outputs}", lambda st, a=a, w=w, o=out, kw=kw: s.linear(a, w, o, stream=st, **kw), out)
    history, length = torch.randint(0, VOCAB, (ROWS, 16), generator=g, device="cuda", dtype=torch.int32), full((ROWS,), 16)
    p = [lily.SamplingParams(presence_penalty=0.5)] * ROWS
    for dtype, out_type in ((F32, F32), (BF16, F32), (BF16, BF16)):
        for rows in (3, 40):
            for pad in (0, 1):
                x = rand(rows, VOCAB, t=dtype)
                out = torch.zeros((rows, VOCAB + pad), dtype=out_type, device="cuda")[:, :VOCAB]
                lists = dict(history_ids=history[:rows], history_len=length[:rows])
                biases = dict(bias_ids=history[:rows, :4].contiguous(), bias_vals=rand(rows, 4), bias_len=full((rows,), 4))
                masks = dict(mask=full((rows, (VOCAB + 31) // 32), 0x55555555))
                for name, params, kw in (("masks", None, masks), ("lists", p[:rows], lists), ("biases", None, biases)):
                    yield (f"adjust {dtype} {out_type} {rows} {pad} {name}", lambda st, x=x, p=params, o=out, kw=kw:
                           s.adjust_logits(x, p, o, stream=st, **kw), out)

free = lambda: torch.cuda.mem_get_info()[0]
scratch = lily.SamplerScratch(VOCAB, max_rows=ROWS, max_history=64, max_list=8)
todo = list(calls(scratch))
stream = torch.cuda.Stream()
torch.cuda.synchronize()
if sys.argv[1] == "memory":
    for name, call, _ in todo:
        before = free()
        call(stream)
        torch.cuda.synchronize()
        assert free() == before, f"{name}: {before - free()} bytes"
else:
    for name, call, out in todo:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(stream)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        captured = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        call(stream)
        torch.cuda.synchronize()
        assert torch.equal(captured.view(torch.uint8) if out.element_size() == 1 else captured.nan_to_num(9.0),
                           out.view(torch.uint8) if out.element_size() == 1 else out.nan_to_num(9.0)), name
        assert out.float().ne(0).any(), name
        del graph
assert scratch.status() == lily.OK
print(len(todo), "calls")
'''


@pytest.mark.parametrize("what", ["memory", "capture"])
def test_first_calls_around_the_head(cuda, lily, what):
    r = subprocess.run([sys.executable, "-c", CHILD, what], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    assert r.stdout.strip().endswith("calls")
