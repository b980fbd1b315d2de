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


def _raises(call):
    try:
        call()
    except IndexError as err:
        return str(err)
    return None


def _bad_ids(rank):
    """Rank 1 asks for ids outside the table; rank 0's are good.  Both raise, and go on afterwards."""
    from hds_b200.band_split import FeatureShards

    shards = FeatureShards(10, 8, rank, WORLD, "cpu", init=table_rows)
    out = []
    for bad in ([2, 10], [2, 2**40], [-1, 3]):
        ids = torch.tensor([1, 6] if rank == 0 else bad)
        out.append(_raises(lambda: shards.dispatch(ids)))
        good = torch.tensor([rank, 5 + rank])
        out.append(torch.equal(shards.dispatch(good), table_rows(0, 10)[good]))
        empty = shards.dispatch(good[:0] if rank else good)
        out.append(tuple(empty.shape) == ((0, 8) if rank else (2, 8)))
    out.append(_raises(shards.check))
    return out


def test_ids_outside_the_table_raise_on_every_rank():
    for result in on_two_ranks(_bad_ids):
        for error, again, empty in zip(result[0:9:3], result[1:9:3], result[2:9:3]):
            assert "outside the table" in error and "[1]" in error
            assert again and empty
        assert result[9] is None


def _different_boundaries(rank):
    """Rank 0 takes rank 1's rows to begin at 5, rank 1 at 6: row 5 has no owner."""
    from hds_b200.band_split import FeatureShards

    shards = FeatureShards(10, 8, rank, WORLD, "cpu", init=table_rows, starts=[0, 5 + rank, 10])
    good = torch.tensor([1, 7])
    out = [_raises(lambda: shards.dispatch(good)) is None]
    shards.dispatch(torch.tensor([5]) if rank == 0 else good)  # met by rank 1, which has no such row
    out.append(_raises(lambda: shards.dispatch(good)))
    out.append(_raises(lambda: shards.dispatch(good)) is None)
    shards.dispatch(torch.tensor([5]) if rank == 0 else good)
    out.append(_raises(shards.check))
    return out


def test_rows_asked_of_a_rank_that_does_not_own_them_are_reported():
    for rank, (first, error, later, checked) in enumerate(on_two_ranks(_different_boundaries)):
        assert first and later
        assert "differ between the ranks" in error and "[1]" in error
        assert (checked is not None) == (rank == 1)


def test_one_rank_indexes_its_rows():
    """Ids that are no rows raise at once on the CPU; gradients of another type are refused."""
    from hds_b200.band_split import FeatureShards

    shards = FeatureShards(10, 8, 0, 1, "cpu", init=table_rows)
    ids = torch.tensor([1, 4, 9])
    assert torch.equal(shards.dispatch(ids), table_rows(0, 10)[ids])
    for _ in range(2):
        shards.combine(ids, torch.ones(8, 3).T)
    want = torch.zeros(10, 8)
    want[ids] = 2
    assert torch.equal(shards.rows.grad, want)
    with pytest.raises(IndexError):
        shards.dispatch(torch.tensor([10]))
