"""Attention of queries that share rows of the cache (b200kv_mla_decode_shared) against 64 bits, on the device."""
import numpy as np
import pytest
import torch

import b200kv
from gpu_util import status_ok, to_dev_i32
from shared_cases import HEADS, LATENT, Case

pytestmark = pytest.mark.gpu


class Call:
    """A case's device arrays; run() is one call into outputs that were NaN."""

    def __init__(self, case, stable=False, quantised=False, q=None):
        self.case, self.stable = case, stable
        pool = case.pool.cuda()
        if case.fused:
            self.cache = (pool,)
        else:
            self.cache = (pool[:, :LATENT].contiguous(), pool[:, LATENT:].contiguous())
        self.view = b200kv.pool_view(*self.cache)
        self.q = case.q.cuda() if q is None else q
        self.table, self.kv_len = to_dev_i32(case.table), to_dev_i32(case.kv_len)
        self.index, self.leader, self.shared = to_dev_i32(case.table_index), to_dev_i32(case.leader), to_dev_i32(case.shared)
        self.out = torch.full((case.batch, case.heads, LATENT), float("nan"), dtype=torch.bfloat16, device="cuda")
        self.lse = torch.full((case.batch, case.heads), float("nan"), dtype=torch.float32, device="cuda")
        self.ws = torch.full((b200kv.decode_shared_workspace_bytes(case.batch, case.heads),), 0xFF, dtype=torch.uint8, device="cuda")
        self.status = b200kv.new_status()
        self.quantised = None
        if quantised:
            self.quantised = (torch.zeros(case.batch, HEADS, LATENT, dtype=torch.uint8, device="cuda"),
                              torch.zeros(case.batch, HEADS, LATENT // 32, dtype=torch.uint8, device="cuda"))

    def run(self, index=True, stream=None):
        b200kv.mla_decode_shared(self.q, self.view, self.table, self.kv_len, self.case.block, self.case.scale, self.leader, self.shared,
                                 table_index=self.index if index else None, out=self.out, lse=self.lse, workspace=self.ws, status=self.status,
                                 stable_tables=self.stable, quantised=self.quantised, stream=stream)
        return self

    def check(self, what=""):
        status_ok(self.status)
        self.case.check(self.out, self.lse, what)


ALONE = [(0, [1]), (0, [63]), (0, [64]), (0, [65]), (0, [127]), (0, [128]), (0, [129]), (0, [0]), (0, [1000])]


@pytest.mark.parametrize("group", ALONE, ids=lambda g: f"len{g[1][0]}")
def test_one_query(group):
    Call(Case([group]).poison_unused()).run().check()


@pytest.mark.parametrize("shared,lens", [
    (64, [64, 64]), (64, [65, 64]), (64, [64, 100]), (128, [128, 128]), (128, [129, 300]), (192, [192, 193]), (256, [700, 256]), (64, [64, 64, 64]),
    (1024, [1025, 1100, 1024, 1500, 1024]), (0, [5, 70]), (0, [0, 3]), (0, [3, 0]), (0, [0, 0]), (128, [1, 0]), (256, [10, 200]), (256, [200, 10, 256, 300]),
    (4096, [4100, 4300]), (6400, [6401] * 7)])
def test_sequences_behind_a_prefix(shared, lens):
    Call(Case([(shared, lens)]).poison_unused()).run().check()


@pytest.mark.parametrize("history,new", [(0, 1), (0, 2), (0, 5), (0, 130), (63, 2), (64, 3), (127, 2), (127, 5), (300, 4), (1000, 9), (5000, 3), (0, 300)])
def test_tokens_of_one_sequence(history, new):
    Call(Case([(history + new, [history + i + 1 for i in range(new)])], one_table=True).poison_unused()).run().check()


@pytest.mark.parametrize("block,fused", [(64, True), (128, False), (192, False), (1024, True)])
def test_several_groups_of_any_shape(block, fused):
    groups = [(block, [block + 1, block + 77]), (0, [5]), (3 * block, [3 * block, 3 * block + 200, 3 * block + 1]), (0, [0]), (2 * block, [10, 2 * block])]
    Call(Case(groups, block=block, fused=fused, gain=3.0).poison_unused(), stable=True).run().check()


@pytest.mark.parametrize("shared_len", [1, 63, 100, 129, 255, 256])
def test_a_shared_length_that_ends_inside_a_tile(shared_len):
    """Whole blocks are common; saying that fewer tokens are is allowed."""
    case = Case([(256, [256, 257, 400])]).poison_unused()
    case.shared = [shared_len] * 3
    Call(case).run().check()


def test_many_queries():
    """More queries than a scan of the list takes at once, some without tokens."""
    rng = np.random.default_rng(5)
    groups = [(int(s) * 64, [int(s) * 64 + int(n) if n > 20 else int(n) for n in rng.integers(0, 90, int(rng.integers(1, 6)))]) for s in rng.integers(0, 3, 200)]
    case = Case(groups).poison_unused()
    assert case.batch > 512
    Call(case).run().check()


def test_without_table_index_a_query_has_its_own_row():
    Call(Case([(128, [130, 200, 128]), (0, [7])]).poison_unused()).run(index=False).check()


def test_a_row_behind_a_query_does_not_reach_it():
    """NaN and infinities in a later token's row stay with the queries that attend over it."""
    for poison in (float("nan"), float("inf")):
        case = Case([(200, [197, 198, 199, 200])], one_table=True)
        case.pool[case.rows_of(3)[199]] = poison
        call = Call(case).run()
        status_ok(call.status)
        assert torch.isnan(call.out[3]).all() or not torch.isfinite(call.out[3].float()).all()
        clean = Case([(200, [197, 198, 199, 200])], one_table=True)
        clean.kv_len[3] = 199
        clean.check(torch.cat([call.out[:3], call.out[2:3] * 0 + clean.want()[0][3:].to(call.out)]), None)


def test_a_nan_in_a_common_row_reaches_every_query():
    case = Case([(640, [640, 700, 641])])
    case.pool[case.rows_of(0)[300]] = float("nan")
    call = Call(case).run()
    status_ok(call.status)
    assert torch.isnan(call.out.float()).all() and torch.isnan(call.lse).all()


def test_growing_scores_rescale():
    """Every step's scores are far above the ones before, in one run and over several."""
    for n in (640, 20000):
        case = Case([(n, [n, n, n])])
        direction = torch.randn(HEADS, 576, generator=torch.Generator().manual_seed(3))[0]
        j = torch.arange(n, dtype=torch.float32) / n * 40
        case.q = (direction + 0.01 * torch.randn(case.q.shape, generator=torch.Generator().manual_seed(4))).to(torch.bfloat16)
        case.pool[torch.from_numpy(case.rows_of(0))] = ((j[:, None] - 20) * direction / 10 + case.pool[torch.from_numpy(case.rows_of(0))].float() * 0.1).to(torch.bfloat16)
        Call(case).run().check(f"{n} tokens")


def test_minus_infinity_scores_have_no_weight():
    """A key of infinities scores -infinity (or NaN); here all queries are positive there and the key is -infinity."""
    case = Case([(128, [128, 200])])
    case.q[..., 575] = 1.0
    case.pool[torch.from_numpy(case.rows_of(0)[5:6]), 575] = -float("inf")
    call = Call(case).run()
    status_ok(call.status)
    keep = [j for j in range(128) if j != 5]
    for b, n in enumerate(case.kv_len):
        rows = np.concatenate([case.rows_of(b)[keep], case.rows_of(b)[128:]])
        k, q = case.pool[torch.from_numpy(rows)].double(), case.q[b].double()
        s = q @ k.T * case.scale
        p = torch.softmax(s, 1)
        off = (call.out[b].double().cpu() - p @ k[:, :LATENT]).abs()
        assert (off <= 2.0 ** -7 * (p @ k[:, :LATENT].abs())).all()
        assert (call.lse[b].double().cpu() - torch.logsumexp(s, 1)).abs().max() < 1e-3


def test_strided_queries():
    case = Case([(128, [130, 200, 128])])
    wide = torch.full((3, HEADS + 3, 600), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, :HEADS, :576] = case.q.cuda()
    Call(case, q=wide[:, :HEADS, :576]).run().check()


def test_queries_laid_out_by_head_and_one_query_for_all():
    case = Case([(128, [130, 200, 128])])
    Call(case, q=case.q.cuda().transpose(0, 1).contiguous().transpose(0, 1)).run().check()
    case.q[:] = case.q[0].clone()
    Call(case, q=case.q[0].cuda()[None].expand(3, -1, -1)).run().check()


def test_rows_that_lie_beyond_32_bits():
    case = Case([(256, [257, 400, 256])]).poison_unused()
    call, before = Call(case), 2 ** 32 // 1152 // case.block + 1
    pool = torch.empty(before * case.block + len(case.pool), 576, dtype=torch.bfloat16, device="cuda")
    pool[before * case.block:] = call.cache[0]
    call.cache, call.view, call.table = (pool,), b200kv.pool_view(pool), call.table + before
    call.run().check()


def test_quantised_output_is_the_quantisers():
    call = Call(Case([(256, [300, 257, 256])]), quantised=True).run()
    call.check()
    codes, scales = torch.zeros_like(call.quantised[0]).view(3, -1), torch.zeros_like(call.quantised[1]).view(3, -1)
    b200kv.mx_quant_e4m3(call.out.view(3, -1), codes, scales)
    assert torch.equal(codes.view_as(call.quantised[0]), call.quantised[0]) and torch.equal(scales.view_as(call.quantised[1]), call.quantised[1])


@pytest.mark.parametrize("heads,block", [(16, 64), (64, 16), (128, 128)])
def test_other_geometries(heads, block):
    case = Case([(128, [130, 200, 128]), (0, [0]), (0, [9])], block=block, heads=heads)
    call = Call(case).run(index=False)
    status_ok(call.status)
    case.check(call.out, call.lse)


def test_bad_table_entries_are_recorded():
    for change in ("block", "negative", "row", "short"):
        case = Case([(256, [300, 300])])
        call = Call(case)
        if change == "block":
            call.table[0, 1] = case.blocks
        elif change == "negative":
            call.table[0, 1] = -1
        elif change == "row":
            call.index[0] = 2
        else:
            call.kv_len[1] = case.table.shape[1] * 64 + 1
        call.run()
        torch.cuda.synchronize()
        assert call.status.tolist()[0] == b200kv.DEV_BAD_BLOCK


def test_lengths_beyond_the_table_end_at_its_first_missing_block():
    """Whatever stands in kv_len: the call ends, says so, and the other queries' results are theirs."""
    for long in (2 ** 31 - 1, 2 ** 30, 129):
        case = Case([(128, [100, 128]), (0, [128]), (0, [60])] * 60).poison_unused()
        call = Call(case)
        call.kv_len[2::4] = long
        call.run()
        torch.cuda.synchronize()
        assert call.status.tolist()[0] == b200kv.DEV_BAD_BLOCK
        want, _, bound, _ = case.want()
        keep = [b for b in range(case.batch) if b % 4 != 2]
        assert ((call.out.double().cpu() - want).abs() <= bound)[keep].all()
    case = Case([(128, [100, 128]), (0, [0])]).poison_unused()
    call = Call(case)
    call.kv_len[2] = -5   # a negative length is an empty one
    call.run().check()


def test_arrays_that_say_nothing_sensible_still_cover_every_query():
    """Leaders that name no group: queries are paired by equal leaders of neighbours only, and each reads its own rows."""
    case = Case([(0, [100]), (0, [70]), (0, [0]), (0, [200]), (0, [300])]).poison_unused()
    case.leader, case.shared = [7, 7, -2, -2, 99], [0, 0, -5, 0, 0]
    Call(case).run().check()


def test_captured_and_replayed_beside_an_eager_call_on_another_stream():
    case, other = Case([(1024, [1025, 1100, 1500])]), Case([(512, [600] * 9)], seed=2)
    call, eager = Call(case), Call(other)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call.run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):
            call.run()
    for _ in range(3):
        call.out.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager.run()
        graph.replay()
        call.check()
        eager.check()


def test_lengths_that_the_kernel_before_wrote():
    """Without stable_tables the arrays may come from the kernel before; with it they may not, the queries and rows still may."""
    case = Case([(1024, [1025, 1100, 1500])])
    for stable in (False, True):
        call = Call(case, stable=stable)
        lens, q = call.kv_len.clone(), call.q.clone()
        for _ in range(5):
            if not stable:
                call.kv_len.zero_()
            call.q.zero_()
            torch.cuda.synchronize()
            call.q.copy_(q)
            if not stable:
                call.kv_len.copy_(lens)
            call.run()
            call.check()


def test_two_calls_give_the_same_bits():
    case = Case([(3000 // 64 * 64, [3100, 3200, 2950, 4000])])
    first, second = Call(case).run(), Call(case).run()
    torch.cuda.synchronize()
    assert torch.equal(first.out, second.out) and torch.equal(first.lse, second.lse)


def test_runs_of_many_items_in_a_workspace_that_the_call_before_reads_too():
    """More items a run than its own list holds (some 35), with stable tables, behind a call of another kind in the same workspace."""
    case, times = Case([(128, [130, 140]), (64, [66, 65]), (0, [3, 3]), (0, [0])] + [(0, [1 + i]) for i in range(9)]).poison_unused(), 200
    want, want_lse, bound, lse_bound = (t.cuda() for t in case.want())
    n, last = case.batch, int(case.leader[-1])
    assert last == n - 1
    many = Call(case, stable=True)
    many.q = many.q.repeat(times, 1, 1)
    many.out, many.lse = many.out.repeat(times, 1, 1), many.lse.repeat(times, 1)
    many.leader = (many.leader[None, :] + n * torch.arange(times, dtype=torch.int32, device="cuda")[:, None]).flatten().contiguous()
    many.kv_len, many.shared, many.index = many.kv_len.repeat(times), many.shared.repeat(times), many.index.repeat(times)
    many.ws = torch.full((b200kv.decode_shared_workspace_bytes(n * times, HEADS),), 0xFF, dtype=torch.uint8, device="cuda")
    before = torch.full((n, HEADS, LATENT), float("nan"), dtype=torch.bfloat16, device="cuda")
    own_rows = torch.stack([many.table[i] for i in case.table_index]).contiguous()
    for _ in range(3):
        b200kv.mla_decode(case.q.cuda(), many.view, own_rows, to_dev_i32(case.kv_len), case.block, case.scale, out=before,
                          workspace=many.ws, status=many.status, stable_tables=True)
        many.run()
    status_ok(many.status)
    assert ((before.double() - want).abs() <= bound).all()
    assert ((many.out.double().view(times, n, HEADS, LATENT) - want).abs() <= bound).all()
    lse, empty = many.lse.double().view(times, n, HEADS), torch.isinf(want_lse)
    assert (lse[:, empty] == -float("inf")).all() and ((lse - want_lse).abs()[:, ~empty] <= lse_bound[~empty]).all()
