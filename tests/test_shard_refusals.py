"""What one rank of a sharded step would refuse, every rank refuses before it waits for the others (gloo, CPU)."""
import os
import socket
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Scratch:
    """Refuses what the library refuses of a shard; notes the rest."""

    def __init__(self):
        self.calls = []

    def adjust_logits(self, logits, params, *, first_id, stream, count_slots=None, **kw):
        import lily_b200 as lily

        if count_slots is not None and first_id != 0:
            raise lily.LilyError(lily.ERR_ARG, "count_slots needs first_id 0")
        self.calls.append("adjust")

    def __getattr__(self, name):
        return lambda *a, **k: self.calls.append(name)


def _worker(rank, world, port, out):
    sys.path.insert(0, ROOT)
    import datetime

    import torch
    import torch.distributed as dist

    import lily_b200 as lily
    import lily_b200.shard as sh

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=20))
    scratch = Scratch()
    args = (scratch, torch.zeros((100, 512), dtype=torch.int8), None, torch.zeros((2, 512)), [lily.SamplingParams()] * 2, None, rank * 100)
    said = []
    for adjust in ({"count_slots": [0, 1]}, {"count_slots": None}):
        try:
            sh.sharded_lmhead_draw(*args, adjust=adjust)
            said.append("drawn")
        except Exception as e:
            said.append(f"{type(e).__name__} {getattr(e, 'code', '')}")
    with open(f"{out}.{rank}", "w") as f:
        f.write("; ".join([*said, *scratch.calls]))
    dist.barrier()
    dist.destroy_process_group()


def test_histogram_slots_of_shards(lily, tmp_path):
    import torch.multiprocessing as mp

    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(2, port, str(tmp_path / "said")), nprocs=2, join=True)
    for rank in range(2):
        assert (tmp_path / f"said.{rank}").read_text() == f"LilyError {lily.ERR_ARG}; drawn; lmhead_logits; adjust; shard_candidates; merge_draw"


def test_one_rank_may_have_them(lily):
    import torch

    import lily_b200.shard as sh

    scratch = Scratch()
    sh.sharded_lmhead_draw(scratch, torch.zeros((100, 512), dtype=torch.int8), None, torch.zeros((2, 512)),
                           [lily.SamplingParams()] * 2, None, 0, adjust={"count_slots": [0, 1]})
    assert scratch.calls == ["lmhead_logits", "adjust", "shard_candidates", "merge_draw"]
