"""Ranks that start at different times are not taken as gone: the first step
waits for them longer than a later one (CPU, processes and a TCPStore)."""
import time

import torch.multiprocessing as mp

from stealcode_b200 import shards
from tests.test_shards import _free_port


def _late_rank(rank, world, port, late, out):
    import datetime

    from torch.distributed import TCPStore

    store = TCPStore("127.0.0.1", port, world, rank == 0, timeout=datetime.timedelta(seconds=30))
    sh = shards.StreamShards(store, rank, world, 100, timeout_s=0.5)
    if rank == late:
        time.sleep(2.0)  # loads its model, say
    try:
        out.put((rank, [sh.step(s) for s in range(2)]))
    except RuntimeError as exc:
        out.put((rank, str(exc)))
    if rank == 0:
        time.sleep(1.0)  # the store's host outlives the other ranks' last reads


def test_a_rank_that_starts_late_is_waited_for():
    for late in (0, 1):
        ctx = mp.get_context("spawn")
        q = ctx.Queue()
        port = _free_port()
        procs = [ctx.Process(target=_late_rank, args=(r, 2, port, late, q)) for r in range(2)]
        for p in procs:
            p.start()
        res = dict(q.get(timeout=120) for _ in procs)
        for p in procs:
            p.join(timeout=60)
            assert p.exitcode == 0
        assert res == {0: [(0, 50, [])] * 2, 1: [(50, 100, [])] * 2}, res
