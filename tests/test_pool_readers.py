"""Calls that only look at a block pool (statistics, the invariant check) beside calls that plan: they share no memory that either
writes, so a thread that watches the pool changes nothing in what another does."""
import threading
import time

import numpy as np
import pytest

import b200kv

SEQS, COLUMNS, BS = 40, 50, 64


@pytest.fixture(scope="module")
def engine():
    e = b200kv.Engine(layers=1, max_seqs=SEQS, num_blocks=SEQS * COLUMNS, block_size=BS, max_blocks_per_seq=COLUMNS, max_step_tokens=SEQS * COLUMNS * BS,
                      scale=1.0 / 24.0, backend=b200kv.ARENA_HOST_SIM)
    rng = np.random.default_rng(3)
    for s in range(SEQS):
        e.admit(s)
        e.begin_step([s], [int(rng.integers(1, COLUMNS * BS))])
        e.end_step()
    for s in range(0, SEQS, 3):
        e.release(s)
    return e


def plan(e):
    moves = np.empty((e.config.num_blocks, 3), dtype=np.int32)
    n = b200kv.lib.b200kv_block_pool_plan_compact(b200kv.lib.b200kv_engine_block_pool(e._h), len(moves), moves.ctypes.data)
    return moves[:n].copy()


@pytest.mark.parametrize("watch", ["statistics", "validate"])
def test_a_watching_thread_does_not_disturb_a_plan(engine, watch):
    pool = b200kv.lib.b200kv_engine_block_pool(engine._h)
    look = engine.stats_json if watch == "statistics" else lambda: b200kv.check(b200kv.lib.b200kv_block_pool_validate(pool))
    want, stop, failed = plan(engine), threading.Event(), []
    assert len(want) > 100 and (want[:, 2] > 0).all()

    def watcher():
        said = engine.stats_json()
        while not stop.is_set():
            try:
                look()
                assert engine.stats_json() == said
            except Exception as e:  # noqa: BLE001
                failed.append(e)
                return

    threads = [threading.Thread(target=watcher) for _ in range(2)]
    for t in threads:
        t.start()
    try:
        until = time.monotonic() + 1.0
        while time.monotonic() < until:
            assert np.array_equal(plan(engine), want)
    finally:
        stop.set()
        for t in threads:
            t.join()
    assert not failed, failed[0]
