"""What attention of queries that share rows asks for beside its arguments: the partials of the runs, however many queries there are."""
import ctypes

import pytest
import torch

import b200kv

PARTIALS = 74 * 2 * 128 * (512 + 2) * 4   # two items a run of 128 rows: the sums, the maximum and the sum of weights in fp32


@pytest.mark.parametrize("batch", [1, 9, 148, 149, 512, 4096, 16384])
def test_the_workspace_does_not_grow_with_the_queries(batch):
    need = b200kv.decode_shared_workspace_bytes(batch)
    assert PARTIALS < need <= PARTIALS + 4096 + 64 * batch   # (an entry of the list of work a query)
    assert need >= b200kv.decode_shared_workspace_bytes(max(1, batch // 2))


def test_the_split_decode_of_other_geometries_still_fits():
    """148 sequences of 128 heads in two parts each; from 149 on a sequence is one part and needs none."""
    at = {batch: b200kv.decode_shared_workspace_bytes(batch, 128) for batch in (9, 148, 149, 16384)}
    assert at[148] >= 148 * 2 * 128 * (512 + 2) * 4 and at[9] >= 9 * 32 * 128 * (512 + 2) * 4
    assert at[16384] <= PARTIALS + 4096 + 64 * 16384


@pytest.mark.gpu
@pytest.mark.parametrize("max_step_tokens", [32, 16384])
def test_an_engine_of_long_chunks_reserves_no_more(max_step_tokens):
    e = b200kv.Engine(layers=1, max_seqs=8, num_blocks=16, block_size=64, max_blocks_per_seq=8, max_step_tokens=max_step_tokens, scale=1.0 / 24.0)
    b200kv.lib.b200kv_arena_workspace_bytes.restype = ctypes.c_int64
    b200kv.lib.b200kv_arena_workspace_bytes.argtypes = [ctypes.c_void_p]
    held = b200kv.lib.b200kv_arena_workspace_bytes(b200kv.lib.b200kv_engine_arena(e._h))
    assert held <= PARTIALS + (1 << 20) + 64 * max_step_tokens


@pytest.mark.gpu
@pytest.mark.parametrize("heads,block,batch,row", [(64, 64, 148, 578), (64, 64, 160, 578), (16, 16, 30, 576), (128, 64, 148, 578), (128, 64, 150, 576)])
def test_other_geometries_run_in_it(heads, block, batch, row):
    """Queries that the tensor cores cannot load (rows of 578 values) and other head counts, many of them."""
    from shared_cases import Case
    from test_gpu_shared import Call

    case = Case([(0, [1 + 7 * i % 90]) for i in range(batch)], block=block, heads=heads).poison_unused()
    wide = torch.zeros(batch, heads, row, dtype=torch.bfloat16, device="cuda")
    wide[..., :576] = case.q.cuda()
    Call(case, q=wide[..., :576]).run(index=False).check()
