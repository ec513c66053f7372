"""Tokens taken back when no block is free: the blocks that the call itself empties are enough for the copy that it needs (host memory
stands for the device's)."""
import ctypes

import numpy as np
import pytest

import b200kv

BS = 64


def engine(num_blocks, **k):
    a = dict(layers=2, max_seqs=4, num_blocks=num_blocks, block_size=BS, max_blocks_per_seq=6, max_step_tokens=300, scale=1.0 / 24.0, backend=b200kv.ARENA_HOST_SIM)
    return b200kv.Engine(**{**a, **k})


def caches(e):
    c, rows = e.cache, e.config.num_blocks * BS
    at = lambda handle, width: np.ctypeslib.as_array(ctypes.cast(e.span_address(handle), ctypes.POINTER(ctypes.c_uint16)),  # noqa: E731
                                                     shape=(e.config.layers, rows, width))
    return at(c.latent_handle, 512), at(c.rope_handle, 64)


def rows(e, s, n):
    t = np.arange(n)
    return e.table()[s][t // BS] * BS + t % BS


def fill(e):
    rng = np.random.default_rng(7)
    for cache in caches(e):
        cache[:] = rng.integers(0, 65536, cache.shape)


def grow(e, s, n):
    e.begin_step([s], [n])
    e.end_step()


def state(e):
    return e.table().tolist(), e.free_list().tolist(), [e.seq_len(s) for s in range(4)], e.stats_json()


@pytest.mark.parametrize("own,back", [(10, 40), (10, 11), (10, 73), (130, 131), (130, 160), (130, 257)])
def test_a_trim_in_a_full_pool_takes_the_blocks_that_it_empties(own, back):
    """Sequence 1 has `own` tokens behind 128 common ones and every block is held; `back` tokens leave it inside a common block."""
    e = engine(2 + (own + BS - 1) // BS)
    e.admit(0)
    grow(e, 0, 128)
    e.fork(0, 1)
    grow(e, 1, own)
    fill(e)
    assert len(e.free_list()) == 0
    left = 128 + own - back
    want = [cache[:, rows(e, 1, left)].copy() for cache in caches(e)]
    common = [cache[:, rows(e, 0, 128)].copy() for cache in caches(e)]
    e.trim(1, back)
    assert e.seq_len(1) == left and e.seq_len(0) == 128
    for cache, mine, theirs in zip(caches(e), want, common):
        assert (cache[:, rows(e, 1, left)] == mine).all() and (cache[:, rows(e, 0, 128)] == theirs).all()
    shared = left // BS
    assert (e.table()[1][:shared] == e.table()[0][:shared]).all() and (left % BS == 0 or e.table()[1][shared] != e.table()[0][shared])
    assert len(e.free_list()) == (own + BS - 1) // BS - (1 if left % BS else 0)
    if left % BS:
        grow(e, 1, 1)   # its half-filled block is its own


def test_a_trim_that_empties_nothing_of_its_own_is_still_refused():
    e = engine(2)
    e.admit(0)
    grow(e, 0, 128)
    e.fork(0, 1)
    before = state(e)
    with pytest.raises(b200kv.B200KVError, match="free"):
        e.trim(1, 1)
    assert state(e) == before
    with pytest.raises(b200kv.B200KVError):
        e.trim(1, 70)   # the block that this gives back is the other's too
    assert state(e) == before
    e.trim(1, 64)


def test_a_copy_that_fails_in_a_full_pool_changes_nothing():
    e = engine(5)
    e.admit(0)
    grow(e, 0, 128)
    e.fork(0, 1)
    grow(e, 1, 130)
    fill(e)
    before, cache = state(e), [c.copy() for c in caches(e)]
    b200kv.fault_inject("b200kv_copy_blocks")
    with pytest.raises(b200kv.B200KVError, match="injected"):
        e.trim(1, 140)
    assert b200kv.fault_clear() == 1 and state(e) == before
    assert all((a == b).all() for a, b in zip(cache, caches(e)))
    e.trim(1, 140)
    grow(e, 0, 1)
    assert e.seq_len(1) == 118 and e.seq_len(0) == 129


def test_random_histories_in_a_small_pool():
    """Forks, growth and trims with hardly a block to spare: what a trim leaves is what was there, and it is refused only when it
    empties no block of its own and none is free."""
    done = 0
    for seed in range(20):
        rng = np.random.default_rng(seed)
        e = engine(7)
        tokens, next_value = {}, 1
        marks = caches(e)[0][0, :, 0]   # a value a row stands for its token
        e.admit(0)
        tokens[0] = []
        for _ in range(120):
            s = int(rng.choice(list(tokens)))
            op = rng.integers(0, 4)
            try:
                if op == 0:
                    n = int(rng.integers(1, 100))
                    grow(e, s, n)
                    at = rows(e, s, len(tokens[s]) + n)[-n:]
                    marks[at] = np.arange(next_value, next_value + n)
                    tokens[s] += list(range(next_value, next_value + n))
                    next_value += n
                elif op == 1 and len(tokens) < 4:
                    d = next(x for x in range(4) if x not in tokens)
                    e.fork(s, d)
                    tokens[d] = list(tokens[s])
                elif op == 2 and len(tokens) > 1:
                    e.release(s)
                    del tokens[s]
                elif op == 3:
                    n = int(rng.integers(0, len(tokens[s]) + 1))
                    table, left = e.table(), len(tokens[s]) - n
                    named = np.concatenate([table[x][:(len(tokens[x]) + BS - 1) // BS] for x in tokens])
                    mine = table[s][:(len(tokens[s]) + BS - 1) // BS]
                    half = left // BS if n and left % BS else None
                    alone = [int((named == b).sum()) == 1 for b in mine]
                    able = half is None or alone[half] or len(e.free_list()) > 0 or any(alone[half + 1:])
                    try:
                        e.trim(s, n)
                    except b200kv.B200KVError:
                        assert not able
                    else:
                        assert able
                        tokens[s] = tokens[s][:left]
                        done += 1
            except b200kv.B200KVError:
                pass   # no block for the growth or the fork
            for x, want in tokens.items():
                assert e.seq_len(x) == len(want) and marks[rows(e, x, len(want))].tolist() == [v % 65536 for v in want]
    assert done > 100
