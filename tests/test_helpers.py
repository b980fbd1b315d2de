"""The support that multi-process tests lean on."""
import time

import pytest

torch = pytest.importorskip("torch")
import torch.multiprocessing as mp

import helpers  # noqa: F401  (the workers import this module, and with it what they wait by)


def _send(queue, kind):
    if kind == "tensors":
        for k in range(3):
            queue.put(torch.full((1000,), float(k)))
    queue.put(kind)


def test_a_worker_stays_until_its_tensors_are_fetched():
    """The parent looks three seconds after the worker has sent its tensors and has nothing else to do."""
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    worker = ctx.Process(target=_send, args=(queue, "tensors"))
    worker.start()
    first = queue.get(timeout=120)
    time.sleep(3.0)
    rest = [queue.get(timeout=60) for _ in range(3)]
    assert all(torch.equal(t, torch.full((1000,), float(k))) for k, t in enumerate([first, *rest[:2]]))
    assert rest[2] == "tensors"
    worker.join(timeout=60)
    assert worker.exitcode == 0
