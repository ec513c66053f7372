"""Sequences that share blocks, on the host: fork, unshare, compact and what they do to grow, ungrow and release, against a model
that keeps every sequence's tokens as values; the engine's calls over host memory; refusals of the device entry points."""
import ctypes

import numpy as np
import pytest
import torch

import b200kv

BS = 4


class Model:
    """Each live sequence as the list of its tokens' values, and the pool's rows as an array."""

    def __init__(self, blocks, seqs, columns):
        self.pool = b200kv.BlockPool(blocks, BS, seqs, columns)
        self.rows = np.full(blocks * BS, -1)
        self.tokens, self.next = {}, 0

    def copy(self, moves):
        before = self.rows.copy()
        for s, d, n in moves:
            self.rows[d * BS:d * BS + n] = before[s * BS:s * BS + n]

    def grow(self, seq, n):
        slots = self.pool.grow(seq, n)
        for slot in slots:
            assert self.pool.ref_count(slot // BS) == 1   # nothing is written where others read
            self.rows[slot] = self.next
            self.tokens[seq].append(self.next)
            self.next += 1

    def check(self):
        self.pool.validate()
        table, lens = self.pool.table(), self.pool.lens()
        named = np.zeros(self.pool.num_blocks, dtype=int)
        for seq, want in self.tokens.items():
            assert lens[seq] == len(want)
            j = np.arange(len(want))
            assert self.rows[table[seq][j // BS] * BS + j % BS].tolist() == want
            named[table[seq][:(len(want) + BS - 1) // BS]] += 1
        assert [self.pool.ref_count(b) for b in range(self.pool.num_blocks)] == named.tolist()
        assert sorted(self.pool.free_list()) == np.flatnonzero(named == 0).tolist()


@pytest.mark.parametrize("seed", range(6))
def test_random_histories(seed):
    rng = np.random.default_rng(seed)
    m = Model(24, 6, 10)
    for _ in range(600):
        live, idle = list(m.tokens), [s for s in range(6) if s not in m.tokens]
        op = rng.integers(0, 7)
        before = (m.pool.table(), m.pool.lens(), m.pool.free_list())
        try:
            if op == 0 and idle:
                m.pool.admit(idle[0])
                m.tokens[idle[0]] = []
            elif op == 1 and live:
                s = int(rng.choice(live))
                left = len(m.tokens[s])
                if left % BS and m.pool.ref_count(int(m.pool.table()[s][left // BS])) > 1:
                    with pytest.raises(b200kv.B200KVError):
                        m.pool.grow(s, 1)
                    m.copy(m.pool.unshare(s, left // BS))
                m.grow(s, int(rng.integers(0, 9)))
            elif op == 2 and live and idle:
                s = int(rng.choice(live))
                n = int(rng.integers(-1, len(m.tokens[s]) + 1))
                m.copy(m.pool.fork(s, idle[-1], n))
                m.tokens[idle[-1]] = m.tokens[s][:] if n < 0 else m.tokens[s][:n]
            elif op == 3 and live:
                s = int(rng.choice(live))
                n = int(rng.integers(0, len(m.tokens[s]) + 1))
                m.pool.ungrow(s, n)
                m.tokens[s] = m.tokens[s][:len(m.tokens[s]) - n]
            elif op == 4 and live and rng.random() < 0.5:
                s = int(rng.choice(live))
                m.pool.release(s)
                del m.tokens[s]
            elif op == 5:
                moves = m.pool.plan_compact(int(rng.integers(-1, 6)))
                assert len({*moves[:, 0], *moves[:, 1]}) == 2 * len(moves)   # no block twice
                m.copy(moves)
                m.pool.apply_moves(moves)
            elif op == 6 and live:
                s = int(rng.choice(live))
                if m.tokens[s]:
                    m.copy(m.pool.unshare(s, int(rng.integers(0, (len(m.tokens[s]) + BS - 1) // BS))))
        except b200kv.B200KVError:   # refused for want of blocks or columns: nothing changed
            now = (m.pool.table(), m.pool.lens(), m.pool.free_list())
            assert all((a == b).all() for a, b in zip(before, now))
        m.check()
    moves = m.pool.plan_compact()
    m.copy(moves)
    m.pool.apply_moves(moves)
    m.check()
    used = m.pool.num_blocks - m.pool.free_count
    assert m.pool.free_list().tolist() == list(range(used, m.pool.num_blocks))


def test_refusals_of_the_pool():
    pool = b200kv.BlockPool(3, BS, 4, 3)
    pool.admit(0)
    pool.grow(0, 10)   # all three blocks, the last half filled
    for call in (lambda: pool.fork(0, 1), lambda: pool.fork(0, 0), lambda: pool.fork(1, 2), lambda: pool.fork(0, 1, 11), lambda: pool.fork(0, 1, -2),
                 lambda: pool.fork(0, 9), lambda: pool.unshare(0, 3), lambda: pool.unshare(0, -1), lambda: pool.unshare(1, 0),
                 lambda: pool.apply_moves([[0, 1, 4]]), lambda: pool.apply_moves([[3, 0, 4]]), lambda: pool.ungrow(0, 11)):
        before = (pool.table(), pool.lens(), pool.free_list())
        with pytest.raises(b200kv.B200KVError):
            call()
        assert all((a == b).all() for a, b in zip(before, (pool.table(), pool.lens(), pool.free_list())))
        pool.validate()
    assert len(pool.fork(0, 1, 8)) == 0 and pool.ref_count(0) == 2   # whole blocks need none
    pool.ungrow(1, 1)
    with pytest.raises(b200kv.B200KVError, match="unshare"):
        pool.grow(1, 1)
    with pytest.raises(b200kv.B200KVError):
        pool.unshare(1, 1)   # no free block
    assert pool.ref_count(3) == -1 and len(pool.unshare(0, 2)) == 0 and len(pool.plan_compact(0)) == 0


def engine(**k):
    a = dict(layers=2, max_seqs=4, num_blocks=12, block_size=64, max_blocks_per_seq=4, max_step_tokens=8, scale=1.0 / 24.0, backend=b200kv.ARENA_HOST_SIM)
    return b200kv.Engine(**{**a, **k})


def caches(e):
    c, rows = e.cache, e.config.num_blocks * e.config.block_size
    at = lambda handle, width: np.ctypeslib.as_array(ctypes.cast(e.span_address(handle), ctypes.POINTER(ctypes.c_uint16)),  # noqa: E731
                                                     shape=(e.config.layers, rows, width))
    return at(c.latent_handle, 512), at(c.rope_handle, 64)


def test_engine_forks_trims_and_compacts_over_host_memory():
    e = engine(max_step_tokens=300)
    latent, rope = caches(e)
    e.admit(0)
    e.begin_step([0], [130])
    e.end_step()
    table = e.table()
    rng = np.random.default_rng(1)
    latent[:] = rng.integers(0, 65536, latent.shape)
    rope[:] = rng.integers(0, 65536, rope.shape)
    rows = lambda s, n: e.table()[s][np.arange(n) // 64] * 64 + np.arange(n) % 64  # noqa: E731
    want = latent[:, rows(0, 130)].copy(), rope[:, rows(0, 130)].copy()

    def same(s, n):
        return (latent[:, rows(s, n)] == want[0][:, :n]).all() and (rope[:, rows(s, n)] == want[1][:, :n]).all()

    e.fork(0, 1)
    assert e.seq_len(1) == 130 and (e.table()[1][:2] == table[0][:2]).all() and e.table()[1][2] != table[0][2] and same(1, 130)
    e.fork(1, 2, 128)
    assert e.seq_len(2) == 128 and same(2, 128)
    e.trim(2, 30)   # its second block is common: a copy of its own before anything is written there
    assert e.seq_len(2) == 98 and e.table()[2][1] not in (table[0][1], 0) and same(2, 98) and same(0, 130)
    e.trim(1, 2)    # down to whole blocks: nothing to copy
    e.begin_step([2, 1, 0])
    e.end_step()
    e.release(0)
    assert e.compact(1) == 1 and e.compact() >= 0
    used = {int(b) for s in (1, 2) for b in e.table()[s][:(e.seq_len(s) + 63) // 64]}
    assert used == set(range(len(used))) and same(1, 128) and same(2, 98)
    assert e.compact() == 0 and e.compact(0) == 0
    for call in (lambda: e.fork(0, 3), lambda: e.fork(1, 2), lambda: e.trim(1, 1000), lambda: e.trim(0, 1), lambda: e.trim(1, -1)):
        with pytest.raises(b200kv.B200KVError):
            call()
    e.begin_step([1])
    for call in (lambda: e.fork(1, 3), lambda: e.trim(1, 1), lambda: e.compact()):
        with pytest.raises(b200kv.B200KVError, match="in flight"):
            call()
    e.abort_step()


def test_shared_tokens_count_once_in_the_statistics():
    e = engine(max_step_tokens=300)
    tokens = lambda: int(e.stats_json().split('"active_context_tokens": ')[1].split(",")[0])  # noqa: E731
    e.admit(0)
    e.begin_step([0], [130])
    e.end_step()
    assert tokens() == 130
    e.fork(0, 1)          # 128 are common, the two behind them copied
    assert tokens() == 132
    e.begin_step([1, 0], [3, 1])
    assert tokens() == 136
    e.abort_step()
    assert tokens() == 132
    e.release(0)
    assert tokens() == 130
    e.trim(1, 30)
    assert tokens() == 100


def test_a_copy_that_fails_changes_nothing():
    e = engine(max_step_tokens=300)
    e.admit(0)
    e.begin_step([0], [100])
    e.end_step()
    e.admit(1)
    e.begin_step([1], [65])
    e.end_step()
    e.release(0)
    e.fork(1, 2, 64)
    state = lambda: (e.table().tolist(), e.free_list().tolist(), [e.seq_len(s) for s in range(4)], e.stats_json())  # noqa: E731
    for call in (lambda: e.fork(1, 3), lambda: e.trim(2, 1), lambda: e.compact()):
        before = state()
        b200kv.fault_inject("b200kv_copy_blocks")
        with pytest.raises(b200kv.B200KVError, match="injected"):
            call()
        assert b200kv.fault_clear() == 1 and state() == before
    e.trim(2, 1)
    assert e.compact() > 0


def test_a_step_of_several_tokens_or_of_forks_uploads_its_queries():
    e = engine(layers=1, max_step_tokens=10, num_blocks=200, max_blocks_per_seq=150, max_seqs=5)
    queries = lambda: np.ctypeslib.as_array(ctypes.cast(e.span_address(0), ctypes.POINTER(ctypes.c_int32)), shape=(4, 10)).copy()  # noqa: E731
    e.admit(0)
    e.admit(1)
    e.begin_step([1, 0], [3, 2])
    assert queries()[:, :5].tolist() == [[1, 2, 3, 1, 2], [0, 0, 0, 3, 3], [3, 3, 3, 2, 2], [0, 0, 0, 1, 1]]
    e.end_step()
    e.release(1)
    for _ in range(900):   # (ten tokens a step)
        e.begin_step([0], [10])
        e.end_step()
    for s in (1, 2, 3):
        e.fork(0, s)
    e.admit(4)
    e.begin_step([4, 0, 1, 2, 3])
    whole = 9002 // 64 * 64   # (two tokens of the first step, nine hundred times ten)
    got = queries()
    assert got[:, :5].tolist() == [[1] + [9003] * 4, [0, 1, 1, 3, 3], [0] + [whole] * 4, [0, 1, 2, 3, 4]]
    e.end_step()


def test_find_shared():
    table = [[3, 4, 5, 0], [3, 4, 6, 7], [3, 4, 5, 0], [3, 9, 5, 1], [8, 9, 5, 1], [8, 9, 0, 0], [2, 9, 0, 0]]
    lens = [12, 13, 11, 16, 16, 8, 8]
    leader, shared = b200kv.find_shared(table, lens, 4)
    assert leader.tolist() == [0, 0, 2, 2, 4, 4, 6] and shared.tolist() == [8, 8, 4, 4, 8, 8, 0]
    leader, shared = b200kv.find_shared(np.zeros((2, 3)), [100, 7], 4)   # lengths beyond the table; a half-filled block does not count
    assert leader.tolist() == [0, 0] and shared.tolist() == [4, 4]
    leader, shared = b200kv.find_shared(np.zeros((0, 3)), [], 4)
    assert len(leader) == 0
    with pytest.raises(b200kv.B200KVError):
        b200kv.find_shared(table, lens, 0)


STREAM = type("Stream", (), {"cuda_stream": 0})
BF16, I32 = torch.bfloat16, torch.int32


def _shared(**k):
    a = dict(q=torch.zeros(2, 64, 576, dtype=BF16), view=b200kv.pool_view(torch.zeros(128, 576, dtype=BF16)), block_table=torch.zeros(2, 1, dtype=I32),
             kv_len=torch.zeros(2, dtype=I32), block_size=64, scale=1.0 / 24.0, leader=torch.zeros(2, dtype=I32), shared_len=torch.zeros(2, dtype=I32),
             out=torch.zeros(2, 64, 512, dtype=BF16), workspace=torch.zeros(b200kv.decode_shared_workspace_bytes(2), dtype=torch.uint8))
    b200kv.mla_decode_shared(**{**a, **k}, stream=STREAM)


@pytest.mark.parametrize("change,code", [
    (dict(kv_len=None), b200kv.ERR_NULLPTR), (dict(leader=None), b200kv.ERR_NULLPTR), (dict(shared_len=None), b200kv.ERR_NULLPTR), (dict(out=None), b200kv.ERR_NULLPTR),
    (dict(workspace=None), b200kv.ERR_NULLPTR), (dict(workspace=torch.zeros(64, dtype=torch.uint8)), b200kv.ERR_INVALID),
    (dict(block_size=0), b200kv.ERR_INVALID), (dict(block_size=48), b200kv.ERR_INVALID), (dict(scale=0.0), b200kv.ERR_INVALID), (dict(scale=-1.0), b200kv.ERR_INVALID),
    (dict(scale=float("nan")), b200kv.ERR_INVALID),
    (dict(block_table=torch.zeros(1, 1, dtype=I32)), b200kv.ERR_INVALID),   # a row per query without table_index
    (dict(out=torch.zeros(2 * 64 * 512 + 1, dtype=BF16)[1:]), b200kv.ERR_INVALID),
    (dict(q=torch.zeros(2, 16, 576, dtype=BF16), table_index=torch.zeros(2, dtype=I32)), b200kv.ERR_INVALID),
    (dict(block_size=32, table_index=torch.zeros(2, dtype=I32)), b200kv.ERR_INVALID),
    (dict(quantised=(torch.zeros(1, dtype=torch.uint8), None)), b200kv.ERR_INVALID)])
def test_refusals_of_shared_attention(change, code):
    with pytest.raises(b200kv.B200KVError) as refused:
        _shared(**change)
    assert refused.value.code == code


def test_an_empty_batch_needs_nothing():
    _shared(q=torch.zeros(0, 64, 576, dtype=BF16), kv_len=None, leader=None, shared_len=None, out=None, workspace=None)
    assert b200kv.decode_shared_workspace_bytes(0) == 0 and b200kv.decode_shared_workspace_bytes(-1) == 0


def _copy(view=None, moves=torch.zeros(2, 3, dtype=I32), block_size=64, **k):
    b200kv.copy_blocks(b200kv.pool_view(torch.zeros(128, 576, dtype=BF16)) if view is None else view, moves, block_size, stream=STREAM, **k)


@pytest.mark.parametrize("change", [dict(block_size=0), dict(block_size=-64), dict(block_size=48), dict(layers=-1), dict(layers=2),
                                    dict(layers=2, latent_layer_stride=4, rope_layer_stride=8), dict(layers=2, latent_layer_stride=8, rope_layer_stride=-8)])
def test_refusals_of_copy_blocks(change):
    with pytest.raises(b200kv.B200KVError) as refused:
        _copy(**change)
    assert refused.value.code == b200kv.ERR_INVALID


def test_copies_of_nothing_need_no_device():
    _copy(moves=torch.zeros(0, 3, dtype=I32))
    _copy(layers=0)
    view = b200kv.pool_view(torch.zeros(128, 576, dtype=BF16))
    assert b200kv.lib.b200kv_copy_blocks(ctypes.byref(view), 1, 0, 0, None, 2, 64, None, None) == b200kv.ERR_NULLPTR


@pytest.mark.parametrize("call,name", [(_shared, "b200kv_mla_decode_shared"), (_copy, "b200kv_copy_blocks")])
def test_injected_failures(call, name):
    b200kv.fault_inject(name)
    with pytest.raises(b200kv.B200KVError, match="injected"):
        call()
    assert b200kv.fault_clear() == 1
