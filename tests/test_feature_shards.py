"""FeatureShards over two gloo ranks on the CPU: what it takes, and how it reports ids outside its rows."""
import os
import socket

import pytest

torch = pytest.importorskip("torch")
import torch.multiprocessing as mp

WORLD = 2


def free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def table_rows(start, end, channels=8):
    return torch.arange(start * channels, end * channels, dtype=torch.float32).view(-1, channels)


def _worker(rank, port, job, queue):
    import datetime

    import torch.distributed as dist

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=WORLD, timeout=datetime.timedelta(seconds=60))
    try:
        try:
            queue.put((rank, job(rank)))
        except Exception as err:
            queue.put((rank, err))
            raise
        dist.barrier()
    finally:
        dist.destroy_process_group()


def on_two_ranks(job):
    """job(rank) on both ranks; its results (plain values) by rank."""
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    port = free_port()
    procs = [ctx.Process(target=_worker, args=(r, port, job, queue)) for r in range(WORLD)]
    for p in procs:
        p.start()
    out = dict(queue.get(timeout=120) for _ in range(WORLD))
    for result in out.values():
        if isinstance(result, Exception):
            raise result
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    return [out[r] for r in range(WORLD)]


def _combine_types(rank):
    from hds_b200.band_split import FeatureShards

    out = {}
    for dtype in (torch.float32, torch.bfloat16, torch.float16, torch.int32):
        shards = FeatureShards(10, 8, rank, WORLD, "cpu", init=table_rows)
        ids = torch.tensor([1, 4, 7]) + rank
        shards.dispatch(ids)
        shards.combine(ids, torch.full((3, 8), 3 + rank).to(dtype))
        out[str(dtype)] = shards.rows.grad.tolist()
    shards = FeatureShards(10, 8, rank, WORLD, "cpu", init=table_rows)
    shards.dispatch(ids)
    try:
        shards.combine(ids, torch.ones(3, 8, dtype=torch.float64))
        out["float64"] = "taken"
    except (RuntimeError, IndexError):
        out["float64"] = "refused"
    return out


def test_gradients_of_fewer_bits_are_promoted():
    """Rows of 16 bits (or whole numbers) add into the fp32 gradients; 64 bits, which would round, do not."""
    ranks = on_two_ranks(_combine_types)
    want = torch.zeros(10, 8)
    for r in range(WORLD):
        want[torch.tensor([1, 4, 7]) + r] += 3 + r
    for dtype in ("torch.float32", "torch.bfloat16", "torch.float16", "torch.int32"):
        assert torch.equal(torch.tensor(ranks[0][dtype] + ranks[1][dtype]), want), dtype
    assert ranks[0]["float64"] == ranks[1]["float64"] == "refused"
