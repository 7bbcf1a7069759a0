"""The comparators of bench.py's N > 1 line when a rank cannot set one up (a buffer that cannot be exported or opened, a
barrier page that does not appear): EVERY rank has to come back, the root with a note in the figure's place, and the ranks
have to be in step for the next collective.  Two gloo ranks on the CPU; what touches the device is replaced here."""
import os
import sys
import types
from datetime import timedelta

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from conftest import ROOT

WORLD = 2


class _Piece:
    """A shared buffer or barrier whose making fails on the rank it is told to fail on."""
    open_pieces = 0

    def __init__(self, fails, *_, **__):
        if fails:
            raise RuntimeError("refused here")
        self.handle, self.ptr = b"\0" * 64, 4096
        _Piece.open_pieces += 1

    def close(self):
        _Piece.open_pieces -= 1


def _rank_main(rank, port, figure, failing_rank, failing_piece, results):
    if ROOT not in sys.path:
        sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    import bench
    # (a rank left alone in a collective gives up after this long, where the bench's own limit is half an hour)
    dist.init_process_group("gloo", rank=rank, world_size=WORLD, timeout=timedelta(seconds=20))
    mine = rank == failing_rank
    capi = types.SimpleNamespace(
        SharedHostVector=lambda *a, **k: _Piece(mine and failing_piece == "buffer", *a, **k),
        SharedResult=lambda *a, **k: _Piece(mine and failing_piece == "buffer", *a, **k),
        HostBarrier=lambda *a, **k: _Piece(mine and failing_piece == "barrier", *a, **k))
    ctx = {"torch": torch, "dist": dist, "capi": capi, "args": bench.parse_args([]), "world": WORLD, "rank": rank, "ncol": 10,
           "displs": [0, 5], "s_main": None, "shard": None, "stat_dev": torch.device("cpu")}
    try:
        fig = getattr(bench, figure)(ctx)
        after = [None] * WORLD
        dist.all_gather_object(after, ("after", rank))
        results[rank] = (fig, after, _Piece.open_pieces)
    except Exception as e:   # noqa: BLE001  (reported by the parent)
        results[rank] = (f"raised: {e}"[:300], None, None)
    dist.destroy_process_group()


@pytest.mark.parametrize("failing_piece", ["buffer", "barrier"])
@pytest.mark.parametrize("failing_rank", [0, 1])
@pytest.mark.parametrize("figure", ["host_gather_figure", "direct_gather_figure"])
def test_a_rank_that_cannot_set_up_leaves_no_other_rank_waiting(figure, failing_rank, failing_piece):
    port = 31500 + os.getpid() % 2000
    ctx = mp.get_context("spawn")
    with ctx.Manager() as manager:
        results = manager.dict()
        procs = [ctx.Process(target=_rank_main, args=(r, port, figure, failing_rank, failing_piece, results))
                 for r in range(WORLD)]
        for pr in procs:
            pr.start()
        for pr in procs:
            pr.join(timeout=90)
        alive = [pr for pr in procs if pr.is_alive()]
        for pr in alive:
            pr.kill()
            pr.join()
        got = dict(results)
    assert not alive, got
    assert sorted(got) == list(range(WORLD)), got
    for rank in range(WORLD):
        fig, after, still_open = got[rank]
        assert after == [("after", r) for r in range(WORLD)], got            # the ranks are in step
        assert still_open == 0, got                                          # what was opened is closed again
        if rank == 0:
            assert fig["value"] is None and fig["note"] == "not measured: refused here"
        else:
            assert fig is None
