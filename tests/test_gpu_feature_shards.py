"""FeatureShards on the GPU between two ranks that share it: the rows travel over gloo, through the host, so
neither rank's kernels wait for the other's.  The kernels' gather and add, the fetch on a side stream, and the
reports of ids outside the owners' rows."""

import pytest

torch = pytest.importorskip("torch")

import helpers  # noqa: F401
from test_feature_shards import WORLD, _raises, on_two_ranks, table_rows

pytestmark = pytest.mark.gpu

N = 6000


def _steps(rank):
    from hds_b200 import native
    from hds_b200.band_split import FeatureShards

    out = []
    for channels in (24, 13):
        full = table_rows(0, N, channels).cuda()
        gen = torch.Generator().manual_seed(rank)
        ids = torch.randperm(N, generator=gen)[:2500 + rank].sort().values.cuda()
        owner = torch.arange(N) % 3 % WORLD
        for how in (dict(init=lambda a, b: full[a:b]), dict(init=lambda a, b: full[a:b], starts=[0, 100, N]),
                    dict(init=lambda g: full[g], owner=owner)):
            shards = FeatureShards(N, channels, rank, WORLD, "cuda", **how)
            mine = torch.arange(N, device="cuda")
            mine = mine[owner.cuda() == rank] if "owner" in how else mine[shards.start:shards.end]
            out.append(torch.equal(shards.dispatch(ids), full[ids]))
            finish = shards.dispatch_async(ids)
            out.append(torch.equal(finish(), full[ids]))
            grad = torch.full((ids.numel(), channels), rank + 1.0, device="cuda")
            shards.combine(ids, grad.to(torch.bfloat16))
            shards.combine(ids, grad)
            want = torch.zeros(N, channels, device="cuda")
            for r in range(WORLD):
                theirs = torch.randperm(N, generator=torch.Generator().manual_seed(r))[:2500 + r].sort().values.cuda()
                want[theirs] += 2 * (r + 1)
            out.append(torch.equal(shards.rows.grad, want[mine]))
            out.append(_raises(shards.check) is None and native.device_status() == 0)
    return out


def test_dispatch_and_combine_on_the_gpu():
    for result in on_two_ranks(_steps):
        assert result == [True] * 24


def _bad(rank):
    from hds_b200.band_split import FeatureShards

    out = []
    good = torch.tensor([1, 7, 4000], device="cuda")
    shards = FeatureShards(N, 8, rank, WORLD, "cuda", init=table_rows)
    for bad in ([2, N], [-1, 2], [3, 2**40]):
        for call in (shards.dispatch, shards.dispatch_async):
            out.append(_raises(lambda: call(torch.tensor(bad, device="cuda") if rank else good)) is not None)
            out.append(torch.equal(shards.dispatch(good), table_rows(0, N).cuda()[good]))
    # Row 3000 has no owner: rank 0 takes rank 1's block to begin at 3000, rank 1 at 3001.
    shards = FeatureShards(N, 8, rank, WORLD, "cuda", init=table_rows, starts=[0, 3000 + rank, N])
    for call in (shards.dispatch, lambda ids: shards.dispatch_async(ids)()):
        call(torch.tensor([3000], device="cuda") if rank == 0 else good)
        out.append(_raises(lambda: shards.dispatch(good)) is not None)
        out.append(_raises(lambda: shards.dispatch(good)) is None)
    call(torch.tensor([3000], device="cuda") if rank == 0 else good)
    out.append((_raises(shards.check) is not None) == (rank == 1))
    return out


def test_ids_outside_raise_on_every_rank_on_the_gpu():
    for result in on_two_ranks(_bad):
        assert result == [True] * 17
